// One step of beam search (c4s_beam_step, include/c4s_batch.h).
//
// The logits are read once. A wave has a slice of a row and goes through it in
// chunks of 1024 values, 16 a lane: a lane keeps the running maximum and sum of
// exp, and leaves each chunk's largest value in LDS. Of a row's tokens only the
// slice's `width` best can win, since within a row totals are ordered as the logits
// are: the width-th largest of the lanes' maxima bounds them from below, and where a
// lane's chunk reaches that bound (a few do) its 16 values are read once more, 16 such
// sets at a time, and ranked into a list. A list that is full raises the bound.
// The last workgroup of a group to arrive joins the slices' sums (in the slices'
// order). Its threads look at the slices' first places alone: the width-th best of a
// wave's threads' best bounds what can win, and the few places that reach the bound
// are ranked together. 24 groups of 8 rows of 151936, bf16: 27.7 us; when it was 25.5, the slices
// took 18 (8.8 in the mean, memory and VALU together; 58 MB alone would take 10; why the last
// end so late is not known) and the join 7.6. 64 of 4 of 8194, fp32: 13.7, a chain of waits.
// A second kernel brings the states into their new order, a thread a column: it
// reads that of all rows before it writes one, so that outputs may be the inputs.
// (In the first kernel's last workgroups it was a chain of waits: 9 us of 33 for 64
// groups of 4 with 1757 words a row, 40 of 85 for 24 of 8 with 5348.)
//
// Logits that differ can have one total: beside a score of -1e30 all have, and so have some far smaller than the row's
// largest. Where a list's last place is such a one, the tied tokens are looked for once more (to know that takes up to
// 0.4 us).
// Orders are on (value, index) pairs, equal values by the lower index, so results
// do not depend on how rows are cut, but for the sums' rounding. An exponential is one of 32
// bits: exp(z - m) as 2^((z - m) log2 e) is off by 2^-22.8 |z - m| + 2^-23 of itself, least where it
// counts most. A chunk's 16 are added in pairs (2^-22), and all that follows, the chunks' sums and
// what scales them when the maximum rises, is in 64 bits. (One running sum in 32 bits, up to 512 additions
// that may all round the same way, was off by 1.4e-5, and 24 groups of 8 rows of 151936, bf16, without states, took 26.3 us for
// 27.6; with the library's exp for the scaling 28.2.)
// (One fused operation, z log2 e - m log2 e, would save a tenth of the VALU's work and
// overflow on a row whose logits are all the type's lowest value.)

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
constexpr int kMostChunks = 32;                // of a slice
constexpr int kQueue = 128;                    // a lane's chunks that wait to be looked at
constexpr int kFound = 1024;                   // places that are ranked together
constexpr int kStats = 2;                      // words of a part in front of its keys
constexpr float kLog2e = 1.4426950408889634f;

struct BeamArgs {
  c4s_beam a;
  int slices, chunks;    // of a row; chunks of a slice
  int wgs;               // workgroups of a group
  uint32_t* arrived;     // [n_groups]
  int state_wgs;         // workgroups of a group's states
  int32_t* joined;       // [rows] the token that joins a row's history, -1: none; with states
  uint64_t* parts;       // [rows][slices][kStats + width]: maximum, sum (in 64 bits), keys
};

__device__ __forceinline__ void wave_order() {   // this wave's writes to LDS before its reads behind it
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
__device__ __forceinline__ int lanes_before(uint64_t mask, int lane) { return __popcll(mask & ((1ull << lane) - 1)); }

// A token's value as it ranks in its row: larger is better, equal values by the lower token; 0: no token.
__device__ __forceinline__ uint64_t token_key(float z, int v) { return (uint64_t)fkey(z) << 32 | (uint32_t)~v; }
__device__ __forceinline__ float key_value(uint64_t k) { return kfloat((uint32_t)(k >> 32)); }
__device__ __forceinline__ int key_token(uint64_t k) { return (int)~(uint32_t)k; }

// The same of a total: its bits in an order that unsigned numbers have, and the lower (beam, token) first.
struct Total {
  uint64_t t;
  uint32_t at;   // ~(beam * vocab + token)
  __device__ __forceinline__ bool beats(const Total& o) const { return (t > o.t) | ((t == o.t) & (at > o.at)); }
};
constexpr uint64_t kTotalNegInf = 0x000FFFFFFFFFFFFFull;
__device__ __forceinline__ Total no_total() { return Total{0, 0}; }
__device__ __forceinline__ Total total_of(double t, int at) {   // what is not a number counts as -inf, so that all totals have an order
  const uint64_t u = (uint64_t)__double_as_longlong(t + 0.0);   // one zero
  return Total{t == t ? (u >> 63 ? ~u : u | 1ull << 63) : kTotalNegInf, (uint32_t)~at};
}
__device__ __forceinline__ double total_value(const Total& x) {
  return __longlong_as_double((long long)(x.t >> 63 ? x.t ^ 1ull << 63 : ~x.t));
}

// exp y, y <= 0 (below -700, where it no longer counts, 2^-1010): 2^n exp r with |r| up to log 2 / 2, whose series'
// first missing term is r^9 / 9! < 2e-10.
__device__ __forceinline__ double exp_below(double y) {
  const double x = y > -700.0 ? y * 1.4426950408889634 : -1010.0;
  const double n = rint(x), r = (x - n) * 0.6931471805599453;
  double p = 1.0 / 40320.0;
  p = fma(p, r, 1.0 / 5040.0);
  p = fma(p, r, 1.0 / 720.0);
  p = fma(p, r, 1.0 / 120.0);
  p = fma(p, r, 1.0 / 24.0);
  p = fma(p, r, 1.0 / 6.0);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  return ldexp(p, (int)n);
}

// A number that at least n of the wave's lanes reach, and the n-th largest of them but for its last bits (0: fewer
// lanes have one). Twenty bits from the top: a comparison, a count of lanes and a choice each.
__device__ __forceinline__ uint32_t nth_largest(uint32_t v, int n) {
  uint32_t at = 0;
#pragma unroll
  for (int b = 31; b >= 12; --b) {
    const uint32_t up = at | 1u << b;
    at = __popcll(__ballot(v >= up)) >= n ? up : at;
  }
  return at;
}

// The first `most` of list[0 .. n), in order, at its front; n up to 128. One wave's.
__device__ __forceinline__ void keep_best(uint64_t* list, int n, int most, int lane) {
  wave_order();
  const uint64_t a = lane < n ? list[lane] : 0, b = 64 + lane < n ? list[64 + lane] : 0;
  int pa = lane < n ? 0 : most, pb = 64 + lane < n ? 0 : most;
  for (int j = 0; j < n; j += 4) {   // four reads on their way (behind n there may be anything)
    uint64_t o[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = list[j + k];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (j + k >= n) o[k] = 0;
      pa += o[k] > a;
      pb += o[k] > b;
    }
  }
  wave_order();
  if (pa < most) list[pa] = a;
  if (pb < most) list[pb] = b;
  wave_order();
}

// 16 bytes of logits, in memory that is aligned for one.
template <class T>
struct alignas(sizeof(T)) Some {
  T v[16 / sizeof(T)];
};

// A row's logits after penalty and temperature.
template <bool BF16>
struct Logits {
  using T = std::conditional_t<BF16, uint16_t, float>;
  static constexpr int kSome = 16 / sizeof(T), kSets = kPer / kSome;   // values of a load; loads of a lane and chunk
  const T* x;
  const uint32_t* hist;   // null: nothing to penalise
  float pen, temp;

  __device__ __forceinline__ Logits(const c4s_beam& a, int64_t row) {
    x = static_cast<const T*>(a.logits) + row * a.ld;
    pen = a.rep_penalty ? a.rep_penalty[row] : 1.0f;
    temp = a.temperature ? a.temperature[row] : 1.0f;
    hist = pen != 1.0f ? a.hist_bits + row * ((a.vocab + 31) / 32) : nullptr;
    if (!(temp > 0.0f)) temp = 1.0f;
  }
  // Tokens v .. v + kSome - 1, v a multiple of that, as they are in memory; what lies behind `end` is not read.
  __device__ __forceinline__ Some<T> raw(int v, int end) const {
    Some<T> r{};
    if (v + kSome <= end) {
      r = *reinterpret_cast<const Some<T>*>(x + v);
    } else {
#pragma unroll
      for (int j = 0; j < kSome; ++j)
        if (v + j < end) r.v[j] = x[v + j];
    }
    return r;
  }
  __device__ __forceinline__ uint32_t bits(int v, int end) const { return hist && v < end ? hist[v >> 5] >> (v & 31) : 0; }
  __device__ __forceinline__ void value(const Some<T>& r, uint32_t bits, float* z) const {
#pragma unroll
    for (int j = 0; j < kSome; ++j) {
      if constexpr (BF16) z[j] = __uint_as_float((uint32_t)r.v[j] << 16);
      else z[j] = r.v[j];
    }
    if (hist) {
#pragma unroll
      for (int j = 0; j < kSome; ++j) z[j] = bits >> j & 1 ? (z[j] < 0.0f ? z[j] * pen : z[j] / pen) : z[j];
    }
    if (temp != 1.0f) {
#pragma unroll
      for (int j = 0; j < kSome; ++j) z[j] = z[j] / temp;
    }
  }
};

template <bool BF16>
__global__ __launch_bounds__(kBeamThreads, 4) void k_beam(BeamArgs f) {
  __shared__ __align__(16) union {
    struct {
      uint64_t list[kBeamWaves][128];
      uint32_t tops[kBeamWaves][kMostChunks][64];   // keys of the lanes' largest values by chunk
      uint16_t queue[kBeamWaves][kQueue];           // chunk * 64 + lane
    } wave;
    Total found[kFound];
    struct {
      int32_t token[kBeamWidth][kBeamWidth];   // of each row the lowest that tie for the last places
      int32_t n[kBeamWidth];
    } ties;
  } lds;
  __shared__ Total won[kBeamWidth];
  __shared__ uint32_t bounds[kBeamWaves];
  __shared__ double logs[kBeamWidth];                    // the rows' log sum exp(z - tops)
  __shared__ float score[kBeamWidth], tops[kBeamWidth];
  __shared__ int n_found, merged;
  __shared__ uint8_t done[kBeamWidth];
  const c4s_beam& a = f.a;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, W = a.width, V = a.vocab;
  const int group = blockIdx.x / f.wgs, units = W * f.slices, unit = blockIdx.x % f.wgs * kBeamWaves + wave;
  const int64_t row0 = (int64_t)group * W;
  const int words = kStats + W;

  if (unit < units) {
    const int64_t row = row0 + unit / f.slices;
    const int slice = unit % f.slices;
    const Logits<BF16> x(a, row);
    using T = typename Logits<BF16>::T;
    constexpr int kSome = Logits<BF16>::kSome, kSets = Logits<BF16>::kSets;
    const int begin = slice * f.chunks * kChunk, end = min(begin + f.chunks * kChunk, V);
    // value kSome i + j of the lane: token v0 + 64 kSome i + kSome lane + j; two chunks are on their way
    Some<T> ahead[2][kSets];
    uint32_t ahead_bits[2][kSets];
    auto token = [&](int v0, int i, int l) { return v0 + 64 * kSome * i + kSome * l; };
    auto load = [&](int which, int v0) {
#pragma unroll
      for (int i = 0; i < kSets; ++i) {
        ahead[which][i] = x.raw(token(v0, i, lane), end);
        ahead_bits[which][i] = x.bits(token(v0, i, lane), end);
      }
    };
    load(0, begin);
    if (begin + kChunk < end) load(1, begin + kChunk);
    const bool idle = (a.done && a.done[row]) || a.score[row] == -__builtin_inff();   // its logits do not matter
    if (!idle) {
      uint32_t (*chunk_tops)[64] = lds.wave.tops[wave];
      float m = -__builtin_inff();
      double sum = 0.0;
      uint32_t most = 0;   // key of the lane's largest value; 0: it has none
      float z[kPer];
      auto chunk = [&](int which, int v0, int at) {
#pragma unroll
        for (int i = 0; i < kSets; ++i) x.value(ahead[which][i], ahead_bits[which][i], z + kSome * i);
        if (v0 + 2 * kChunk < end) load(which, v0 + 2 * kChunk);
        if (v0 + kChunk > end) {
#pragma unroll
          for (int i = 0; i < kPer; ++i)
            if (token(v0, i / kSome, lane) + i % kSome >= end) z[i] = -__builtin_inff();   // adds nothing
        }
        float top = z[0];
#pragma unroll
        for (int i = 1; i < kPer; ++i) top = fmaxf(top, z[i]);
        const uint32_t key = token(v0, 0, lane) < end ? fkey(top) : 0;
        chunk_tops[at][lane] = key;
        most = max(most, key);
        if (top > m) {
          sum *= exp_below((double)m - (double)top);
          m = top;
        }
        if (m > -__builtin_inff()) {
          float e[kPer];
#pragma unroll
          for (int i = 0; i < kPer; ++i) e[i] = __builtin_amdgcn_exp2f((z[i] - m) * kLog2e);
#pragma unroll
          for (int n = kPer / 2; n; n /= 2)
#pragma unroll
            for (int i = 0; i < n; ++i) e[i] += e[i + n];
          sum += (double)e[0];
        } else {
#pragma unroll
          for (int i = 0; i < kPer; ++i) sum = z[i] != z[i] ? (double)z[i] : sum;   // NaN among the logits is NaN here
        }
      };
      for (int v0 = begin, at = 0; v0 < end; v0 += 2 * kChunk, at += 2) {
        chunk(0, v0, at);
        if (v0 + kChunk < end) chunk(1, v0 + kChunk, at + 1);
      }
      // what a place in the list takes at least: the W-th largest of the lanes' values (0: not so many lanes have one)
      const uint32_t bound = nth_largest(most, W);
      uint64_t* list = lds.wave.list[wave];
      uint16_t* queue = lds.wave.queue[wave];
      int kept = 0, waiting = 0;
      uint64_t least = 0;   // a full list's last place
      auto add = [&](uint64_t key, int& n) {   // one of each lane
        const bool take = key > least && (uint32_t)(key >> 32) >= bound;
        const uint64_t some = __ballot(take);
        if (n + __popcll(some) > 128) {   // no room: what there is, ranked
          keep_best(list, n, W, lane);
          n = min(n, W);
          if (n == W) least = list[W - 1];
        }
        if (take) list[n + lanes_before(some, lane)] = key;
        n += __popcll(some);
      };
      auto rank = [&](int n) {
        keep_best(list, n, W, lane);
        kept = min(n, W);
        if (kept == W) least = list[W - 1];
      };
      constexpr int kAtOnce = 64 / kSets;
      if (begin + kChunk >= end) {   // one chunk: its values are still here
        int n = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const int v = token(begin, i / kSome, lane) + i % kSome;
          add(v < end ? token_key(z[i], v) : 0, n);
        }
        rank(n);
      } else {
        wave_order();
        for (int v0 = begin, at = 0; v0 < end; v0 += kChunk, ++at) {
          const uint32_t top = chunk_tops[at][lane];
          // (the highest key that the lane's values may have)
          const bool reaches = top >= bound && top != 0 && (kept < W || token_key(kfloat(top), v0) > least);
          const uint64_t in = __ballot(reaches);
          if (reaches) queue[waiting + lanes_before(in, lane)] = (uint16_t)(at * 64 + lane);
          waiting += __popcll(in);
          const bool last = v0 + kChunk >= end;
          // as many lanes' values as a wave reads at once, kSets lanes each
          while (waiting >= kAtOnce || (last && waiting)) {
            wave_order();
            const int now = min(waiting, kAtOnce);
            const int what = lane / kSets < now ? queue[lane / kSets] : -1;
            const int move = now + lane < waiting ? queue[now + lane] : 0, move2 = now + 64 + lane < waiting ? queue[now + 64 + lane] : 0;
            const int v = token(begin + (what >> 6) * kChunk, lane % kSets, what & 63);
            float y[kSome];
            if (what >= 0) x.value(x.raw(v, end), x.bits(v, end), y);
            wave_order();
            if (now + lane < waiting) queue[lane] = (uint16_t)move;
            if (now + 64 + lane < waiting) queue[64 + lane] = (uint16_t)move2;
            waiting -= now;
            int n = kept;
#pragma unroll
            for (int j = 0; j < kSome; ++j) add(what >= 0 && v + j < end ? token_key(y[j], v + j) : 0, n);
            rank(n);
          }
        }
      }
      // the slice's maximum, sum and list
      const float top = wave_max_dpp(m);
      const double s = wave_sum_dpp(m == top ? sum : sum * exp_below((double)m - (double)top));
      uint64_t* part = f.parts + (row * f.slices + slice) * words;
      uint64_t w = 0;
      if (lane < kept) w = list[lane];
      if (lane < W) __hip_atomic_store(part + kStats + lane, w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (lane == 0) {
        __hip_atomic_store(part, (uint64_t)__float_as_uint(top), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(part + 1, (uint64_t)__double_as_longlong(s), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    }
  }
  if (!last_to_arrive(f.arrived + group, f.wgs)) return;

  // What this needs of memory is asked for at once: a thread's slice's first places, the sums.
  const uint64_t* parts = f.parts + row0 * f.slices * words;
  auto word = [&](int u, int i) { return __hip_atomic_load(parts + (int64_t)u * words + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
  const int tid = threadIdx.x;
  uint64_t first[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) first[i] = tid < units && i < W ? word(tid, kStats + i) : 0;
  // A wave has every fourth row; of up to 64 slices all sums are on their way.
  constexpr int kRowsOfWave = kBeamWidth / kBeamWaves;
  float most[kRowsOfWave];
  double part[kRowsOfWave];
  auto stats = [&](int i, int j, int s) {
    const bool there = j < W && s < f.slices;
    most[i] = there ? __uint_as_float((uint32_t)word(j * f.slices + s, 0)) : -__builtin_inff();
    part[i] = there ? __longlong_as_double((long long)word(j * f.slices + s, 1)) : 0.0;
  };
#pragma unroll
  for (int i = 0; i < kRowsOfWave; ++i) stats(i, wave + kBeamWaves * i, lane);
  if (tid < W) {
    score[tid] = a.score[row0 + tid];
    done[tid] = a.done ? a.done[row0 + tid] : 0;
  }
  if (tid == 0) n_found = merged = 0;
#pragma unroll
  for (int i = 0; i < kRowsOfWave; ++i) {
    const int j = wave + kBeamWaves * i;
    if (j >= W) break;   // (of a row whose logits do not matter, whatever there is)
    float m = -__builtin_inff();
    double sum = 0.0;
    for (int s0 = 0; s0 < f.slices; s0 += 64) {
      if (s0) stats(i, j, s0 + lane);
      const float t = fmaxf(m, wave_max_dpp(most[i]));
      const double more = wave_sum_dpp(most[i] == t ? part[i] : part[i] * exp_below((double)most[i] - (double)t));
      sum = (m == t ? sum : sum * exp_below((double)m - (double)t)) + more;
      m = t;
    }
    if (lane == 0) {
      tops[j] = m;
      logs[j] = sum == 0.0 ? 0.0 : log(sum);
    }
  }
  __syncthreads();

  auto lost = [&](int j) { return !(score[j] > -__builtin_inff()) | (logs[j] != logs[j]); };   // all of row j's totals are -inf
  auto total_at = [&](int j, float z, int v) {
    return total_of(z == -__builtin_inff() ? -__builtin_inf() : (double)score[j] + (((double)z - (double)tops[j]) - logs[j]), j * V + v);
  };
  // Place `at` of slice u, whose key is k where the row's logits matter.
  auto total = [&](int u, int at, uint64_t k) {
    const int j = u / f.slices;
    if (done[j]) return u == j * f.slices && at == 0 ? total_of(score[j], j * V + a.stop_token) : no_total();
    if (lost(j)) return u == j * f.slices && at < V ? total_of(-__builtin_inf(), j * V + at) : no_total();
    return k ? total_at(j, key_value(k), key_token(k)) : no_total();
  };
  // Whether the slice whose last place this is may have left out lower tokens of the same total: its logit's total is
  // that of the next lower number too.
  auto merges = [&](int u, uint64_t k, const Total& t) {
    const int j = u / f.slices;
    return !done[j] && !lost(j) && key_value(k) > -__builtin_inff() && total_at(j, kfloat((uint32_t)(k >> 32) - 1), 0).t == t.t;
  };
  Total* found = lds.found;
  {
    Total mine = no_total();
    for (int u = tid; u < units; u += kBeamThreads) {
      const Total t = total(u, 0, u < kBeamThreads ? first[0] : word(u, kStats));
      if (t.beats(mine)) mine = t;
    }
    // (of a total's bits the upper half: a bound a little lower does as well)
    const uint32_t of_wave = nth_largest((uint32_t)(mine.t >> 32), W);
    if (lane == 0) bounds[wave] = of_wave;
  }
  __syncthreads();
  const uint32_t bound = max(max(bounds[0], bounds[1]), max(bounds[2], bounds[3]));
  static_assert(kBeamWaves == 4, "the waves' bounds");
  for (int u = tid; u < units; u += kBeamThreads) {
    for (int at0 = 0; at0 < W; at0 += 4) {   // places are in order: behind one that does not reach the bound none does
      uint64_t k[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) k[i] = at0 == 0 && u < kBeamThreads ? first[i] : (at0 + i < W ? word(u, kStats + at0 + i) : 0);
      bool more = true;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const Total t = at0 + i < W ? total(u, at0 + i, k[i]) : no_total();
        more = more && t.at && (uint32_t)(t.t >> 32) >= bound;
        if (more) {
          const int n = atomicAdd(&n_found, 1);
          if (n < kFound) found[n] = t;
          if (at0 + i == W - 1 && merges(u, k[i], t)) merged = 1;
        }
      }
      if (!more) break;
    }
  }
  __syncthreads();
  if (n_found <= kFound) {
    const int n = n_found;
    for (int i = tid; i < n; i += kBeamThreads) {
      const Total mine = found[i];
      int at = 0;
      for (int o = 0; o < n; o += 4) {
        Total x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = found[min(o + k, kFound - 1)];
#pragma unroll
        for (int k = 0; k < 4; ++k) at += (o + k < n) & x[k].beats(mine);
      }
      if (at < W) won[at] = mine;
    }
  } else {
    // too many places reach the bound (lists whose totals hardly differ): the best, the best behind it, and so on
    Total last = no_total();
    for (int i = 0; i < W; ++i) {
      Total mine = no_total();
      for (int u = threadIdx.x; u < units; u += kBeamThreads)
        for (int at = 0; at < W; ++at) {
          const Total t = total(u, at, word(u, kStats + at));
          if (!t.at || t.t < mine.t) break;
          if ((i == 0 || last.beats(t)) && t.beats(mine)) mine = t;
        }
      __syncthreads();
      found[threadIdx.x] = mine;
      __syncthreads();
      for (int d = kBeamThreads / 2; d; d /= 2) {
        if ((int)threadIdx.x < d && found[threadIdx.x + d].beats(found[threadIdx.x])) found[threadIdx.x] = found[threadIdx.x + d];
        __syncthreads();
      }
      last = found[0];
      if (threadIdx.x == 0) won[i] = last;
      __syncthreads();
    }
  }
  __syncthreads();
  if (merged) {
    // Of different logits with equal totals a slice's list has the highest logits, but the lowest tokens come first. The last
    // place's total is right, and so are the places above it, of which a list leaves out none: the row's tokens with that
    // very total, looked for in all its logits, fill the others. A wave takes every fourth row. (This is seldom, and slow
    // where ties are few: 0.5 ms for a row of 151936 bf16, 3 us for one of 8194.)
    const uint64_t tie = won[W - 1].t;
    for (int j = wave; j < W; j += kBeamWaves) {
      int32_t* tied = lds.ties.token[j];
      int n = 0;
      if (done[j]) {
        n = total_of(score[j], 0).t == tie;
        if (n && lane == 0) tied[0] = a.stop_token;
      } else if (lost(j)) {
        n = tie == kTotalNegInf ? min(W, V) : 0;
        if (lane < n) tied[lane] = lane;
      } else {
        const Logits<BF16> x(a, row0 + j);
        constexpr int kSome = Logits<BF16>::kSome;
        for (int v0 = 0; v0 < V && n < W; v0 += 64 * kSome) {
          const int v = v0 + kSome * lane;
          float z[kSome];
          x.value(x.raw(v, V), x.bits(v, V), z);
          int before = n;   // those of the lanes before
          uint32_t mine = 0;
#pragma unroll
          for (int i = 0; i < kSome; ++i) {
            const bool same = v + i < V && total_at(j, z[i], 0).t == tie;
            const uint64_t some = __ballot(same);
            before += lanes_before(some, lane);
            n += __popcll(some);
            mine |= same ? 1u << i : 0u;
          }
#pragma unroll
          for (int i = 0; i < kSome; ++i) {
            const int place = before + __popc(mine & ((1u << i) - 1));
            if ((mine >> i & 1) && place < W) tied[place] = v + i;
          }
        }
      }
      if (lane == 0) lds.ties.n[j] = min(n, W);
    }
    __syncthreads();
    if (tid == 0) {
      int at = 0;
      while (won[at].t > tie) ++at;
      for (int j = 0; j < W; ++j)
        for (int i = 0; i < lds.ties.n[j] && at < W; ++i) won[at++] = Total{tie, ~(uint32_t)(j * V + lds.ties.token[j][i])};
    }
    __syncthreads();
  }
  if (tid < W) {
    const Total t = won[tid];
    const int at = (int)~t.at, parent = at / V, token = at - parent * V;
    const int64_t r = row0 + tid;
    a.out_parent[r] = parent;
    a.out_token[r] = token;
    a.out_score[r] = (float)total_value(t);
    if (a.out_done) a.out_done[r] = done[parent] || token == a.stop_token;
    if (f.joined) f.joined[r] = done[parent] || token == a.stop_token ? -1 : token;
  }
}

// A workgroup has a group's rows over 256 columns of the history and the states, in this order.
__global__ __launch_bounds__(kBeamThreads) void k_beam_states(BeamArgs f) {
  __shared__ uint32_t column[kBeamWidth][kBeamThreads];
  __shared__ int parents[kBeamWidth], tokens[kBeamWidth];
  const c4s_beam& a = f.a;
  const int tid = threadIdx.x, W = a.width;
  const int64_t row0 = (int64_t)(blockIdx.x / f.state_wgs) * W;
  int64_t c = (int64_t)(blockIdx.x % f.state_wgs) * kBeamThreads + tid;
  const uint32_t* src = nullptr;
  uint32_t* dst = nullptr;
  int64_t ld_src = 0, ld_dst = 0;
  int hist = -1;   // the word of the history that this is
  if (a.hist_bits) {
    const int64_t words = (a.vocab + 31) / 32;
    if (c < words) {
      src = a.hist_bits + c, dst = a.out_hist_bits + c;
      ld_src = ld_dst = words;
      hist = (int)c;
    }
    c -= words;
  }
  for (int i = 0; i < a.n_states; ++i) {
    const c4s_beam_state& s = a.states[i];
    if (c >= 0 && c < s.words) {
      src = static_cast<const uint32_t*>(s.src) + c, dst = static_cast<uint32_t*>(s.dst) + c;
      ld_src = s.ld_src, ld_dst = s.ld_dst;
    }
    c -= s.words;
  }
  if (tid < W) {
    parents[tid] = a.out_parent[row0 + tid];
    tokens[tid] = f.joined[row0 + tid];
  }
  if (src) {
    for (int j0 = 0; j0 < W; j0 += 8) {   // eight rows' reads on their way
      uint32_t v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = src[(row0 + min(j0 + j, W - 1)) * ld_src];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j0 + j < W) column[j0 + j][tid] = v[j];
    }
  }
  __syncthreads();
  if (!src) return;
  for (int j = 0; j < W; ++j) {
    uint32_t v = column[parents[j]][tid];
    if (hist >= 0 && tokens[j] >= 0 && tokens[j] / 32 == hist) v |= 1u << (tokens[j] % 32);
    dst[(row0 + j) * ld_dst] = v;
  }
}

// How a row is cut: into slices for twelve waves a CU together, of 1 to kMostChunks chunks. In us, for 8 / 12 / 16 / 24
// waves a CU (with sums in 32 bits): 24 groups of 8 rows of 151936 bf16 27.2 / 26.2 / 27.4 / 35.4, fp32 30.8 / 31.0 / 32.5 / 39.9; 192 rows
// 24.3 / 20.7 / 21.1 / 26.8; 256 groups of 4 of 32000 25.1 / 23.4 / 23.2 / 30.3.
BeamArgs beam_args(const c4s_beam& a) {
  BeamArgs f{};
  f.a = a;
  const int64_t rows = (int64_t)a.n_groups * a.width, chunks = (a.vocab + kChunk - 1) / kChunk;
  const int64_t slices = std::max(std::min(std::max<int64_t>(12 * 256 / rows, 1), chunks), (chunks + kMostChunks - 1) / kMostChunks);
  f.chunks = (int)((chunks + slices - 1) / slices);
  f.slices = (int)((chunks + f.chunks - 1) / f.chunks);
  f.wgs = (a.width * f.slices + kBeamWaves - 1) / kBeamWaves;
  int64_t words = a.hist_bits ? (a.vocab + 31) / 32 : 0;
  for (int i = 0; i < a.n_states; ++i) words += a.states[i].words;
  f.state_wgs = (int)((words + kBeamThreads - 1) / kBeamThreads);
  return f;
}

}  // namespace

LayerSpace beam_space(const c4s_beam& a) {
  const BeamArgs f = beam_args(a);
  return {a.n_groups, (int64_t)a.n_groups * a.width * (f.slices * (kStats + a.width) * 2 + 1)};
}

hipError_t launch_beam(const c4s_beam& a, uint32_t* counters, float* space, hipStream_t s) {
  BeamArgs f = beam_args(a);
  f.arrived = counters;
  f.parts = reinterpret_cast<uint64_t*>(space);
  f.joined = f.state_wgs ? reinterpret_cast<int32_t*>(f.parts + (int64_t)a.n_groups * a.width * f.slices * (kStats + a.width)) : nullptr;
  const dim3 grid((unsigned)(a.n_groups * f.wgs)), block(kBeamThreads);
  if (a.dtype == C4S_DTYPE_BF16) hipLaunchKernelGGL(k_beam<true>, grid, block, 0, s, f);
  else hipLaunchKernelGGL(k_beam<false>, grid, block, 0, s, f);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || f.state_wgs == 0) return e;
  hipLaunchKernelGGL(k_beam_states, dim3((unsigned)((int64_t)a.n_groups * f.state_wgs)), block, 0, s, f);
  return hipGetLastError();
}

}  // namespace c4s
