// One step of beam search (c4s_beam_step, include/c4s_batch.h).
//
// The logits are read once. A wave has a slice of a row and goes through it in
// chunks of 1024 values, 16 a lane: it keeps the running maximum and sum of exp a
// lane, and a list in LDS of the slice's `width` best tokens. Of a row's tokens
// only those can win, since within a row totals are ordered as the logits are.
// A chunk costs the list nothing unless a value beats its last place; then a bound
// keeps the newcomers few: of the lanes whose best value does, the width-th best of
// those, which at most width lanes' 16 values reach.
// The last workgroup of a group to arrive joins the slices' sums (64 bits, in the
// slices' order), and takes the group's best from the slices' lists: all lists'
// first places, then all second ones, until a round brings nothing. It then brings
// the states into their new order, a thread a column: it reads that of all rows
// before it writes one, so that outputs may be the inputs.
//
// Orders are on (value, index) pairs, equal values by the lower index, so results
// do not depend on how rows are cut, but for the sums' rounding (2^-24 of a lane's
// part; the totals are 64-bit).

#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "c4s_batch.hpp"
#include "c4s_device.hpp"
#include "c4s_join.hpp"

namespace c4s {
namespace {

constexpr int kBeamThreads = 256, kBeamWaves = kBeamThreads / 64;
constexpr int kPer = 16, kChunk = 64 * kPer;   // values of a lane, and of a wave, at a time

struct BeamArgs {
  c4s_beam a;
  int slices, chunks;    // of a row; chunks of a slice
  int wgs;               // workgroups of a group
  uint32_t* arrived;     // [n_groups]
  uint64_t* parts;       // [rows][slices][2 + width]: maximum, sum, keys
};

__device__ __forceinline__ void wave_order() {   // this wave's writes to LDS before its reads behind it
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
__device__ __forceinline__ uint64_t lane_u64(uint64_t v, int lane) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}

// A token's value as it ranks in its row: larger is better, equal values by the lower token; 0: no token.
__device__ __forceinline__ uint64_t token_key(float z, int v) { return (uint64_t)fkey(z) << 32 | (uint32_t)~v; }
__device__ __forceinline__ float key_value(uint64_t k) { return kfloat((uint32_t)(k >> 32)); }
__device__ __forceinline__ int key_token(uint64_t k) { return (int)~(uint32_t)k; }

// The same of a total.
struct Total {
  double t;
  int32_t at;   // beam * vocab + token; -1: none
  __device__ __forceinline__ bool beats(const Total& o) const { return at >= 0 && (o.at < 0 || t > o.t || (t == o.t && at < o.at)); }
};

template <int N, class T>
struct alignas(sizeof(T)) Row {
  T v[N];
};

template <bool BF16>
__global__ __launch_bounds__(kBeamThreads) void k_beam(BeamArgs f) {
  // A wave's list and its newcomers; the last workgroup's rows and states
  constexpr int kList = kBeamWidth * (kPer + 1);
  __shared__ __align__(16) union {
    uint64_t keys[kBeamWaves][kList];
    struct {
      Total best[kBeamWaves][kBeamWidth + 64];
      double lse[kBeamWidth];
      float score[kBeamWidth];
      uint8_t done[kBeamWidth];
      Total won[kBeamWidth];
      int counts[kBeamWaves];
    } last;
    uint32_t column[kBeamWidth * kBeamThreads];
  } lds;
  __shared__ int parents[kBeamWidth];
  const c4s_beam& a = f.a;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, W = a.width, V = a.vocab;
  const int group = blockIdx.x / f.wgs, units = W * f.slices, unit = blockIdx.x % f.wgs * kBeamWaves + wave;
  const int64_t row0 = (int64_t)group * W;
  const int words = 2 + W;

  if (unit < units) {
    const int64_t row = row0 + unit / f.slices;
    const int slice = unit % f.slices;
    uint64_t* part = f.parts + (row * f.slices + slice) * words;
    const bool idle = (a.done && a.done[row]) || a.score[row] == -__builtin_inff();   // its logits do not matter
    if (!idle) {
      using T = typename std::conditional<BF16, uint16_t, float>::type;
      const T* x = static_cast<const T*>(a.logits) + row * a.ld;
      const uint32_t* hist = a.rep_penalty && a.rep_penalty[row] != 1.0f ? a.hist_bits + row * ((V + 31) / 32) : nullptr;
      const float pen = hist ? a.rep_penalty[row] : 1.0f;
      float temp = a.temperature ? a.temperature[row] : 1.0f;
      if (!(temp > 0.0f)) temp = 1.0f;
      uint64_t* list = lds.keys[wave];
      int kept = 0;
      uint64_t least = 0;   // what a key has to beat
      float m = -__builtin_inff(), sum = 0.0f;
      const int begin = slice * f.chunks * kChunk, end = min(begin + f.chunks * kChunk, V);
      for (int v0 = begin; v0 < end; v0 += kChunk) {
        float z[kPer];   // value 4 i + j of the lane: token v0 + 256 i + 4 lane + j
#pragma unroll
        for (int i = 0; i < kPer / 4; ++i) {
          const int v = v0 + 256 * i + 4 * lane;
          Row<4, T> raw;
          if (v + 4 <= end) {
            raw = *reinterpret_cast<const Row<4, T>*>(x + v);
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) raw.v[j] = v + j < end ? x[v + j] : T();
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if constexpr (BF16) z[4 * i + j] = __uint_as_float((uint32_t)raw.v[j] << 16);
            else z[4 * i + j] = raw.v[j];
          }
          if (hist && v < end) {
            const uint32_t bits = hist[v >> 5] >> (v & 31);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float y = z[4 * i + j];
              if (bits >> j & 1) z[4 * i + j] = y < 0.0f ? y * pen : y / pen;
            }
          }
        }
        if (temp != 1.0f) {
#pragma unroll
          for (int i = 0; i < kPer; ++i) z[i] = z[i] / temp;
        }
        auto token = [&](int i) { return v0 + 256 * (i / 4) + 4 * lane + i % 4; };
        uint64_t best = 0;
        float top = m;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const int v = token(i);
          if (v >= end) {
            z[i] = -__builtin_inff();   // adds nothing
          } else {
            const uint64_t k = token_key(z[i], v);
            best = k > best ? k : best;
            top = fmaxf(top, z[i]);
          }
        }
        if (top > -__builtin_inff()) {
          sum *= expf(m - top);
          m = top;
#pragma unroll
          for (int i = 0; i < kPer; ++i) sum += expf(z[i] - m);
        }
        const uint64_t ask = __ballot(best > least);
        if (!ask) continue;
        uint64_t bound = least;
        if (__popcll(ask) > W) {
          int before = 0;   // lanes whose best is better
#pragma unroll 8
          for (int l = 0; l < 64; ++l) before += lane_u64(best, l) > best;
          const uint64_t at = __ballot(best > least && before == W - 1);
          bound = lane_u64(best, __ffsll((unsigned long long)at) - 1) - 1;
        }
        int n = kept;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const int v = token(i);
          const uint64_t k = v < end ? token_key(z[i], v) : 0;
          const uint64_t in = __ballot(k > bound);
          if (k > bound) list[n + __popcll(in & ((1ull << lane) - 1))] = k;
          n += __popcll(in);
        }
        wave_order();
        // every key's place among all; the first W stay, in order
        uint64_t mine[(kList + 63) / 64];
        int place[(kList + 63) / 64];
#pragma unroll
        for (int c = 0; c < (kList + 63) / 64; ++c) {
          const int i = 64 * c + lane;
          place[c] = W;
          if (64 * c < n && i < n) {
            mine[c] = list[i];
            int p = 0;
            for (int j = 0; j < n; ++j) p += list[j] > mine[c];
            place[c] = p;
          }
        }
        wave_order();
#pragma unroll
        for (int c = 0; c < (kList + 63) / 64; ++c)
          if (place[c] < W) list[place[c]] = mine[c];
        wave_order();
        kept = min(n, W);
        if (kept == W) least = list[W - 1];
        wave_order();
      }
      // the slice's maximum, sum and list
      float top = m;
#pragma unroll
      for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
      double s = top == -__builtin_inff() ? 0.0 : (double)sum * exp((double)m - (double)top);
#pragma unroll
      for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
      uint64_t w = 0;
      if (lane < kept) w = list[lane];
      if (lane < W) __hip_atomic_store(part + 2 + lane, w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (lane == 0) {
        __hip_atomic_store(part, (uint64_t)__float_as_uint(top), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(part + 1, (uint64_t)__double_as_longlong(s), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    }
  }
  if (!last_to_arrive(f.arrived + group, f.wgs)) return;

  auto get = [](const uint64_t* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
  auto& la = lds.last;
  if (threadIdx.x < W) {
    la.score[threadIdx.x] = a.score[row0 + threadIdx.x];
    la.done[threadIdx.x] = a.done ? a.done[row0 + threadIdx.x] : 0;
  }
  __syncthreads();
  for (int j = wave; j < W; j += kBeamWaves) {   // a wave a row
    if (la.done[j] || la.score[j] == -__builtin_inff()) continue;
    const uint64_t* part = f.parts + (row0 + j) * f.slices * words;
    float top = -__builtin_inff();
    for (int s = lane; s < f.slices; s += 64) top = fmaxf(top, __uint_as_float((uint32_t)get(part + (int64_t)s * words)));
#pragma unroll
    for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
    double sum = 0.0;
    if (top > -__builtin_inff())
      for (int s = lane; s < f.slices; s += 64)
        sum += __longlong_as_double((long long)get(part + (int64_t)s * words + 1)) *
               exp((double)__uint_as_float((uint32_t)get(part + (int64_t)s * words)) - (double)top);
#pragma unroll
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    if (lane == 0) la.lse[j] = sum > 0.0 ? (double)top + log(sum) : 0.0;
  }
  __syncthreads();

  // A wave's list from its share of the slices' lists, a place of each a round.
  Total* list = la.best[wave];
  int kept = 0;
  Total least{0.0, -1};
  const Total none{0.0, -1};
  for (int place = 0; place < W; ++place) {
    bool news = false;
    for (int u0 = wave * 64; u0 < units; u0 += kBeamThreads) {
      const int u = u0 + lane;
      Total t = none;
      if (u < units) {
        const int j = u / f.slices, slice = u % f.slices;
        if (la.done[j]) {
          if (slice == 0 && place == 0) t = Total{(double)la.score[j], j * V + a.stop_token};
        } else if (la.score[j] == -__builtin_inff()) {
          if (slice == 0 && place < V) t = Total{-__builtin_inf(), j * V + place};
        } else {
          const uint64_t k = get(f.parts + ((row0 + j) * f.slices + slice) * words + 2 + place);
          if (k) {
            const float z = key_value(k);
            t = Total{z == -__builtin_inff() ? -__builtin_inf() : (double)la.score[j] + ((double)z - la.lse[j]), j * V + key_token(k)};
          }
        }
      }
      if (!(t.t == t.t)) t.t = -__builtin_inf();   // so that all totals have an order
      const bool in = t.beats(kept == W ? least : none);
      const uint64_t ask = __ballot(in);
      if (!ask) continue;
      news = true;
      if (in) list[kept + __popcll(ask & ((1ull << lane) - 1))] = t;
      const int n = kept + __popcll(ask);
      wave_order();
      Total mine[2];
      int at[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int i = 64 * c + lane;
        at[c] = W;
        if (i < n) {
          mine[c] = list[i];
          at[c] = 0;
          for (int o = 0; o < n; ++o) at[c] += list[o].beats(mine[c]);
        }
      }
      wave_order();
#pragma unroll
      for (int c = 0; c < 2; ++c)
        if (at[c] < W) list[at[c]] = mine[c];
      wave_order();
      kept = min(n, W);
      least = list[kept - 1];
      wave_order();
    }
    if (!news) break;   // lists are in order: deeper places are worse
  }
  if (lane == 0) la.counts[wave] = kept;
  __syncthreads();
  {
    // the waves' lists: every total's place among all
    const int i = threadIdx.x % kBeamWidth, w = threadIdx.x / kBeamWidth;
    if (w < kBeamWaves && i < la.counts[w]) {
      const Total mine = la.best[w][i];
      int at = 0;
      for (int o = 0; o < kBeamWaves; ++o)
        for (int p = 0; p < la.counts[o]; ++p) at += la.best[o][p].beats(mine);
      if (at < W) la.won[at] = mine;
    }
  }
  __syncthreads();
  Total won{0.0, 0};
  int parent = 0, token = 0;
  bool was = false;
  if (threadIdx.x < W) {
    won = la.won[threadIdx.x];
    parent = won.at / V;
    token = won.at - parent * V;
    was = la.done[parent];
  }
  __syncthreads();   // (the states' columns lie where the totals did)
  uint32_t* column = lds.column;
  const int cols = kBeamWidth * kBeamThreads / W / kBeamThreads * kBeamThreads;   // columns at a time
  if (threadIdx.x < W) {
    const int64_t r = row0 + threadIdx.x;
    parents[threadIdx.x] = parent;
    a.out_parent[r] = parent;
    a.out_token[r] = token;
    a.out_score[r] = (float)won.t;
    if (a.out_done) a.out_done[r] = was || token == a.stop_token;
  }
  __syncthreads();
  auto carry = [&](const uint32_t* src, int64_t ld_src, uint32_t* dst, int64_t ld_dst, int64_t n) {
    for (int64_t c0 = 0; c0 < n; c0 += cols) {
      for (int c = threadIdx.x; c < cols && c0 + c < n; c += kBeamThreads)
        for (int j = 0; j < W; ++j) column[j * cols + c] = src[(row0 + j) * ld_src + c0 + c];
      for (int c = threadIdx.x; c < cols && c0 + c < n; c += kBeamThreads)
        for (int j = 0; j < W; ++j) dst[(row0 + j) * ld_dst + c0 + c] = column[parents[j] * cols + c];
    }
  };
  for (int i = 0; i < a.n_states; ++i) {
    const c4s_beam_state& s = a.states[i];
    carry(static_cast<const uint32_t*>(s.src), s.ld_src, static_cast<uint32_t*>(s.dst), s.ld_dst, s.words);
  }
  if (a.hist_bits) {
    const int64_t n = (V + 31) / 32;
    carry(a.hist_bits, n, a.out_hist_bits, n, n);
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0x0F70);   // vmcnt(0): the rows are written
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __syncthreads();
    if (threadIdx.x < W && !was && token != a.stop_token) {
      uint32_t* word = a.out_hist_bits + (row0 + threadIdx.x) * n + token / 32;
      *word |= 1u << (token % 32);
    }
  }
}

// How a row is cut: into slices for 4096 waves together, sixteen a CU, of at least a chunk.
BeamArgs beam_args(const c4s_beam& a) {
  BeamArgs f{};
  f.a = a;
  const int64_t rows = (int64_t)a.n_groups * a.width, chunks = (a.vocab + kChunk - 1) / kChunk;
  const int64_t slices = std::min(std::max<int64_t>(4096 / rows, 1), chunks);
  f.chunks = (int)((chunks + slices - 1) / slices);
  f.slices = (int)((chunks + f.chunks - 1) / f.chunks);
  f.wgs = (a.width * f.slices + kBeamWaves - 1) / kBeamWaves;
  return f;
}

}  // namespace

LayerSpace beam_space(const c4s_beam& a) {
  const BeamArgs f = beam_args(a);
  return {a.n_groups, (int64_t)a.n_groups * a.width * f.slices * (2 + a.width) * 2};
}

hipError_t launch_beam(const c4s_beam& a, uint32_t* counters, float* space, hipStream_t s) {
  BeamArgs f = beam_args(a);
  f.arrived = counters;
  f.parts = reinterpret_cast<uint64_t*>(space);
  const dim3 grid((unsigned)(a.n_groups * f.wgs)), block(kBeamThreads);
  if (a.dtype == C4S_DTYPE_BF16) hipLaunchKernelGGL(k_beam<true>, grid, block, 0, s, f);
  else hipLaunchKernelGGL(k_beam<false>, grid, block, 0, s, f);
  return hipGetLastError();
}

}  // namespace c4s
