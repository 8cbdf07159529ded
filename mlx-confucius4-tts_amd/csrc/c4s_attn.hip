// Attention of new tokens over the paged cache (c4s_attn, include/c4s_layers.h).
//
// Both products run transposed, S^T = K Q^T and O^T = V^T P^T, so that a lane
// always holds one row (token, query head; column l % 16 of the results): the
// maximum, the sum and the rescaling are a lane's own, but for two steps across
// the four lanes that share a row. Which positions of a block a matrix row of
// S^T stands for is free; in a block of B positions row 4 g + i of tile t is
// position (B / 4) g + 4 t + i, so that lane group g ends up with the weights of
// B / 4 positions in order, which is what P^T wants of it as the next product's
// operand, and which lie next to each other in a page of the values. Nothing is
// shuffled or transposed in between.

#include <hip/hip_runtime.h>

#include <algorithm>

#include "c4s_join.hpp"
#include "c4s_layers.hpp"

namespace c4s {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

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
    o[i] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);   // the upper halves
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// Keeps what is computed from w behind this place (the conversion of a block's
// codes would otherwise move up to their load, at twice the registers).
__device__ __forceinline__ void here(uint4& w) { asm volatile("" : "+v"(w.x), "+v"(w.y), "+v"(w.z), "+v"(w.w)); }

// Over the four lanes that share a row.
// (v_permlane16_swap exchanges one operand's odd rows of 16 lanes with the
// other's even ones, v_permlane32_swap the halves: of v with itself the two
// results hold v and its partner.)
__device__ __forceinline__ float max4(float v) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float sum4(float v) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Dwords of two bf16, of which those at index lo .. hi - 1 stay and the others become zero.
__device__ __forceinline__ uint4 keep(uint4 w, int at, int lo, int hi) {
  uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int j = at + 2 * i;
    v[i] &= (((j >= lo) & (j < hi)) ? 0xFFFFu : 0u) | (((j + 1 >= lo) & (j + 1 < hi)) ? 0xFFFF0000u : 0u);
  }
  return make_uint4(v[0], v[1], v[2], v[3]);
}

__device__ __forceinline__ bool any_odd(uint4 w) {   // one of eight inf or NaN: the largest exponent there is
  auto e = [](uint32_t v) { return __builtin_bit_cast(u16x2, v & 0x7F807F80u); };
  const u16x2 m = __builtin_elementwise_max(__builtin_elementwise_max(e(w.x), e(w.y)), __builtin_elementwise_max(e(w.z), e(w.w)));
  return max(m[0], m[1]) == 0x7F80u;
}

// The finite halves of w, and ones where the others were.
__device__ __forceinline__ void part_odd(uint32_t& w, uint32_t& odd) {
  odd = ((w & 0x7F80u) == 0x7F80u ? 0x3F80u : 0u) | ((w & 0x7F800000u) == 0x7F800000u ? 0x3F800000u : 0u);
  w &= (odd & 0xFFFFu ? 0u : 0xFFFFu) | (odd >> 16 ? 0u : 0xFFFF0000u);
}

// The rows of one sequence, and what they see.
struct Seq {
  int row0, n_new, past, fst, cap;   // n_new 0: nothing to do
  __device__ __forceinline__ Seq(const AttnArgs& a, int seq) {
    row0 = seq;
    n_new = 1;
    int n = 1;
    if (a.off) {
      row0 = a.off[seq];
      n = a.off[seq + 1] - row0;
      n_new = row0 < 0 ? 0 : min(min(n, a.n_rows - row0), a.max_new);
    } else if (seq >= a.n_rows) {
      n_new = 0;
    }
    past = a.lens[seq] - n;
    cap = a.c.max_pages << a.c.page_shift;
    fst = a.first ? min(max(a.first[seq], 0), cap) : 0;
  }
};

constexpr int kRows = 16;   // rows of a workgroup

// ---- few rows -----------------------------------------------------------------------------
//
// A single token's step reads the cache once and computes next to nothing: what
// counts is how many bytes are on their way. A workgroup has 16 rows of one
// sequence and key head and a chunk of its positions; its four waves take
// blocks of KEYS positions in turn, each with a running maximum and sum of its
// own. Keys and values go from memory straight into the matrix engine's
// registers; a block's keys are asked for as soon as the block before it has
// given its scores, its values as soon as the values before them have been
// used, and its pages are in LDS from the start, so that a wave always has about
// a block in flight and never waits for a table. The waves' parts meet in LDS,
// the chunks' in the workspace, where the last workgroup of a row joins them
// (c4s_join.hpp), in the chunks' order.
//
// The weights enter the second product as bf16 pairs (hi + lo, about 2^-17
// relative), which costs nothing here: rounded once to bf16 they would add an
// error of the size of the output's own rounding.
constexpr int kWaves = 4;
constexpr int kAttnThreads = 64 * kWaves;
constexpr int kMaxParts = 128;       // chunks of a sequence
constexpr int kMaxPages = 1024;      // a chunk's pages, in a table in LDS

struct FewArgs {
  AttnArgs a;
  int chunk, splits, tiles;   // positions a chunk (a multiple of 256); chunks at most; row tiles
  uint32_t* arrived;          // [n_seqs][tiles][key heads]
  float* part;                // [n_seqs][tiles][key heads][splits][kRows][dim + 4]
};

// DH: the head's dims rounded up to 64, 128 or 256; FULL: they are that many.
template <int DH, bool Q8, bool FULL, int KEYS>
__global__ __launch_bounds__(kAttnThreads, DH == 64 ? 3 : (DH == 128 ? 2 : 1)) void k_attn_few(FewArgs f) {
  constexpr int kSteps = DH / 32, kTiles = DH / 16, kNT = KEYS / 16, kOwn = KEYS / 4;   // kOwn: a lane's positions of a block
  constexpr int kKLoads = Q8 ? kNT * kSteps / 2 : kNT * kSteps, kVLoads = Q8 || KEYS == 32 ? kTiles : 2 * kTiles;
  __shared__ float sm[kWaves][kRows], sl[kWaves][kRows];
  __shared__ __align__(16) float so[kWaves][kRows][DH + 4];
  const AttnArgs& a = f.a;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, c = lane % 16, g = lane / 16;
  const int dim = FULL ? DH : a.c.dim;
  // blockIdx.x: (tile, chunk, key head), the heads of one chunk next to each other
  const int head = blockIdx.x % a.c.n_heads, split = blockIdx.x / a.c.n_heads % f.splits, tile = blockIdx.x / a.c.n_heads / f.splits;
  const int seq = blockIdx.y;
  const int shift = a.c.page_shift, ps = 1 << shift;
  // The chunk's part of the table (-1: no page), asked for while the lengths are on their way.
  __shared__ int32_t pages[kMaxPages + 16];
  const int base = split * f.chunk;
  auto fill = [&](int from) {
    const int32_t* table = a.c.table + (int64_t)seq * a.c.table_ld;
    for (int i = threadIdx.x; i < (f.chunk >> shift) + (KEYS >> 4); i += kAttnThreads) {
      const int at = (from >> shift) + i;
      const int p = at < a.c.max_pages ? table[at] : -1;
      pages[i] = p < a.c.n_pages ? p : -1;
    }
  };
  fill(base);
  const Seq sq(a, seq);
  const int n_all = sq.n_new * a.shared, r0 = tile * kRows;
  if (r0 >= n_all) return;
  const int valid = min(kRows, n_all - r0);
  const int r = r0 + min(c, valid - 1);
  auto token_of = [&](int r) { return a.shared == 1 ? r : r / a.shared; };
  const int token = token_of(r), qh = head * a.shared + r - token * a.shared;
  const int lim = min(sq.past + token + 1, sq.cap);                            // this row sees positions before it
  const int least = min(sq.past + token_of(r0) + 1, sq.cap);                  // ... the tile's first row
  const int kend = min(sq.past + token_of(r0 + valid - 1) + 1, sq.cap);     // ... its last
  const int fst = sq.fst;
  const int first_chunk = fst / f.chunk, parts = kend > fst ? (kend - 1) / f.chunk + 1 - first_chunk : 1;
  if (split >= parts) return;
  const int begin = max((first_chunk + split) * f.chunk, fst & ~(KEYS - 1)), end = (int)min((int64_t)(first_chunk + split + 1) * f.chunk, (int64_t)kend);

  uint4 q[kSteps];
  {
    const uint16_t* qp = a.q + (int64_t)(sq.row0 + token) * a.ldq + qh * dim;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      // codes come 16 dims a lane at a time, which are two steps of 8
      const int d = Q8 ? 64 * (s / 2) + 16 * g + 8 * (s % 2) : 32 * s + 8 * g;
      q[s] = FULL || d < dim ? *reinterpret_cast<const uint4*>(qp + d) : make_uint4(0, 0, 0, 0);
    }
  }
  const float c2 = a.scale * kLog2e;
  constexpr int kSize = Q8 ? 1 : 2;
  const uint32_t head_bytes = (uint32_t)(dim * kSize) << shift, page_bytes = head_bytes * (uint32_t)a.c.n_heads;   // below 2^31
  const char* kbase = static_cast<const char*>(a.c.k) + (uint64_t)head_bytes * head + 16 * g + (c % 4) * dim * kSize;
  const char* vbase = static_cast<const char*>(a.c.v) + (uint64_t)head_bytes * head + (uint64_t)(uint32_t)((c * kSize) << shift);
  const uint32_t scale_bytes = 4u * (uint32_t)a.c.n_heads << shift;
  const uint32_t tile_bytes = (16u * kSize) << shift;
  // A block's pages: of the key rows this lane loads, and of the positions it weighs (below 0: none).
  const int origin = (first_chunk + split) * f.chunk >> shift;
  struct Pages { int k, v; };
  auto pages_of = [&](int t) {
    return Pages{pages[((t + kOwn * (c / 4)) >> shift) - origin], pages[((t + kOwn * g) >> shift) - origin]};
  };
  uint4 kr[kKLoads], vr[kVLoads];
  float ks[Q8 ? kOwn : 1], vs[Q8 ? kOwn : 1];
  auto load_keys = [&](int t, const Pages& p) {   // scores of what has no page are dropped
    const uint32_t at = (uint32_t)((t + kOwn * (c / 4)) & (ps - 1)) * (uint32_t)(dim * kSize);
    const char* k = kbase + (uint64_t)(uint32_t)max(p.k, 0) * page_bytes + at;
    constexpr int kRow = kSteps / (Q8 ? 2 : 1);
#pragma unroll
    for (int tt = 0; tt < kNT; ++tt)
#pragma unroll
      for (int st = 0; st < kRow; ++st) {
        int d = 64 * st / (Q8 ? 1 : 2);                                         // dims before this lane's
        if (!FULL && d + (Q8 ? 16 : 8) * g >= dim) d = -(Q8 ? 16 : 8) * g;      // times zeros of q
        kr[tt * kRow + st] = *reinterpret_cast<const uint4*>(k + (4 * tt * dim + d) * kSize);
      }
    if constexpr (Q8) {
      const int vt = t + kOwn * g;
      const char* s = reinterpret_cast<const char*>(a.c.k_scale) + (uint64_t)(uint32_t)max(p.v, 0) * scale_bytes + (uint32_t)(((head << shift) + (vt & (ps - 1))) * 4);
#pragma unroll
      for (int j = 0; j < kOwn; j += 4) *reinterpret_cast<float4*>(&ks[j]) = *reinterpret_cast<const float4*>(s + 4 * j);
    }
  };
  auto load_values = [&](int t, const Pages& p) {
    const uint32_t at = (uint32_t)((t + kOwn * g) & (ps - 1));
    const char* v = vbase + (uint64_t)(uint32_t)max(p.v, 0) * page_bytes + at * kSize;
#pragma unroll
    for (int d = 0; d < kTiles; ++d) {
      if constexpr (Q8) {
        if constexpr (KEYS == 64) vr[d] = *reinterpret_cast<const uint4*>(v);
        else {
          const uint2 w = *reinterpret_cast<const uint2*>(v);
          vr[d] = make_uint4(w.x, w.y, 0, 0);
        }
      } else {
#pragma unroll
        for (int st = 0; st < KEYS / 32; ++st) vr[d * (KEYS / 32) + st] = *reinterpret_cast<const uint4*>(v + 16 * st);
      }
      if (FULL || 16 * (d + 1) < dim) v += tile_bytes;   // tiles behind the last dim are not used
    }
    if constexpr (Q8) {
      const char* s = reinterpret_cast<const char*>(a.c.v_scale) + (uint64_t)(uint32_t)max(p.v, 0) * scale_bytes + ((uint32_t)(head << shift) + at) * 4;
#pragma unroll
      for (int j = 0; j < kOwn; j += 4) *reinterpret_cast<float4*>(&vs[j]) = *reinterpret_cast<const float4*>(s + 4 * j);
    }
  };

  float m = -__builtin_inff(), l = 0.0f;
  f32x4 o[kTiles] = {};
  constexpr int kStride = kWaves * KEYS;
  if (first_chunk) {   // behind padding the chunk is another
    __syncthreads();
    fill((first_chunk + split) * f.chunk);
  }
  __syncthreads();
  int t = begin + wave * KEYS;
  if (t < end) {
    Pages now = pages_of(t);
    load_keys(t, now);
    load_values(t, now);
    for (; t < end; t += kStride) {
      f32x4 s[kNT] = {};
#pragma unroll
      for (int tt = 0; tt < kNT; ++tt)
#pragma unroll
        for (int st = 0; st < kSteps; ++st) {
          uint4 w;
          if constexpr (Q8) {
            uint4 x = kr[tt * (kSteps / 2) + st / 2];
            here(x);
            w = codes(st % 2 ? make_uint2(x.z, x.w) : make_uint2(x.x, x.y));
          } else {
            w = kr[tt * kSteps + st];
          }
          s[tt] = mfma(w, q[st], s[tt]);
          if constexpr (Q8) __builtin_amdgcn_sched_barrier(0);
        }
      __builtin_amdgcn_sched_barrier(0);
      // lane's scores are positions vt .. vt + kOwn - 1 of its row, in order
      const int vt = t + kOwn * g;
      float p[kOwn];
#pragma unroll
      for (int j = 0; j < kOwn; ++j) p[j] = s[j / 4][j % 4] * (Q8 ? c2 * ks[j] : c2);
      const bool there = now.v >= 0;
      const bool edge = t < fst || t + KEYS > min(least, end) || __any(!there);
      const int from = max(fst - vt, 0), to = there ? min(lim, end) - vt : 0;
      auto sees = [&](int j) { return (j >= from) & (j < to); };   // whether this row sees position vt + j
      if (edge) {
#pragma unroll
        for (int j = 0; j < kOwn; ++j) p[j] = sees(j) ? p[j] : -__builtin_inff();
      }
      __builtin_amdgcn_sched_barrier(0);
      // The next block's loads; behind the last block that one's again, whose lines are near (a branch around
      // them would make every wait behind it a wait for all of them).
      const bool more = t + kStride < end;
      const int tn = more ? t + kStride : t;
      const Pages ahead = pages_of(tn);
      load_keys(tn, ahead);
      __builtin_amdgcn_sched_barrier(0);
      float top = p[0];
#pragma unroll
      for (int j = 1; j < kOwn; ++j) top = fmaxf(top, p[j]);
      top = fmaxf(max4(top), m);
      const float base = top == -__builtin_inff() ? 0.0f : top;   // nothing seen yet
      const float old = __builtin_amdgcn_exp2f(m - base);
      m = top;
      l *= old;
#pragma unroll
      for (int d = 0; d < kTiles; ++d) o[d] *= old;
      if constexpr (Q8) {
        if (edge) {   // what is masked may have any scale; what is seen has its own, also at a weight of 0
#pragma unroll
          for (int j = 0; j < kOwn; ++j) vs[j] = sees(j) ? vs[j] : 0.0f;
        }
      }
      uint32_t hi[kOwn / 2], lo[kOwn / 2];
#pragma unroll
      for (int j = 0; j < kOwn; j += 2) {
        float x = __builtin_amdgcn_exp2f(p[j] - base), y = __builtin_amdgcn_exp2f(p[j + 1] - base);
        l += x + y;
        if constexpr (Q8) {
          x *= vs[j];
          y *= vs[j + 1];
        }
        hi[j / 2] = pack(x, y);
        lo[j / 2] = pack(x - low(hi[j / 2]), y - high(hi[j / 2]));
      }
      __builtin_amdgcn_sched_barrier(0);
      auto quad = [](const uint32_t* w) { return make_uint4(w[0], w[1], w[2], w[3]); };
      if constexpr (!Q8) {
        if (edge) {
          // What is not there or not for any row may hold anything: zeros. Where some of the rows see a
          // position and others do not, 0 times a value that is not finite would reach those: such
          // values are taken out, and the rows that see them, at whatever weight, become NaN.
          const int any_to = there ? min(kend, end) - vt : 0;
          int odd = 0;
#pragma unroll
          for (int i = 0; i < kVLoads; ++i) {
            vr[i] = keep(vr[i], 8 * (i % (KEYS / 32)), from, any_to);
            odd |= any_odd(vr[i]);
          }
          if (least != kend && __any(odd)) {
            uint32_t mine[kOwn / 2];   // ones where this row sees
#pragma unroll
            for (int j = 0; j < kOwn; j += 2) mine[j / 2] = (sees(j) ? 0x3F80u : 0u) | (sees(j + 1) ? 0x3F800000u : 0u);
#pragma unroll
            for (int d = 0; d < kTiles; ++d) {
              f32x4 seen = {};
#pragma unroll
              for (int st = 0; st < KEYS / 32; ++st) {
                uint4& v = vr[d * (KEYS / 32) + st];
                uint4 ones;
                part_odd(v.x, ones.x);
                part_odd(v.y, ones.y);
                part_odd(v.z, ones.z);
                part_odd(v.w, ones.w);
                seen = mfma(ones, quad(mine + 4 * st), seen);
              }
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (seen[i] != 0.0f) o[d][i] = __builtin_nanf("");
            }
          }
        }
      }
#pragma unroll
      for (int d = 0; d < kTiles; ++d) {
#pragma unroll
        for (int st = 0; st < KEYS / 32; ++st) {
          uint4 v;
          if constexpr (Q8) {
            v = vr[d];
            here(v);
            v = codes(st ? make_uint2(v.z, v.w) : make_uint2(v.x, v.y));
          }
          else v = vr[d * (KEYS / 32) + st];
          o[d] = mfma(v, quad(hi + 4 * st), o[d]);
          o[d] = mfma(v, quad(lo + 4 * st), o[d]);
        }
        if constexpr (Q8) __builtin_amdgcn_sched_barrier(0);
      }
      __builtin_amdgcn_sched_barrier(0);
      load_values(tn, ahead);
      now = ahead;
    }
  }

  // The waves' parts: of output quad (row, dims 4 i ..) by the thread that has it.
  l = sum4(l);
  if (g == 0) {
    sm[wave][c] = m;
    sl[wave][c] = l;
  }
#pragma unroll
  for (int d = 0; d < kTiles; ++d) *reinterpret_cast<f32x4*>(&so[wave][c][16 * d + 4 * g]) = o[d];
  __syncthreads();
  const int quads = dim / 4;   // a row
  const int64_t group = ((int64_t)seq * f.tiles + tile) * a.c.n_heads + head;
  const int words = kRows * (quads + 1);   // quads a part: the rows', then (maximum, sum) of each row
  float* mine = f.part + (group * f.splits + split) * words * 4;
  auto finish = [&](int row, int i, f32x4 v, float top, float sum) {
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    const int rr = r0 + row, tk = token_of(rr), tok = sq.row0 + tk, hh = head * a.shared + rr - tk * a.shared;
    *reinterpret_cast<uint2*>(a.out + (int64_t)tok * a.ld_out + hh * dim + 4 * i) = make_uint2(pack(v[0] * inv, v[1] * inv), pack(v[2] * inv, v[3] * inv));
    if (a.lse && i == 0) a.lse[(int64_t)tok * a.n_heads + hh] = sum == 0.0f ? -__builtin_inff() : (top + log2f(sum)) * kLn2;
  };
  for (int e = threadIdx.x; e < valid * quads; e += kAttnThreads) {
    const int row = e / quads, i = e % quads;
    float top = sm[0][row];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) top = fmaxf(top, sm[w][row]);
    const float base = top == -__builtin_inff() ? 0.0f : top;
    float sum = 0.0f;
    f32x4 v = {};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float fw = __builtin_amdgcn_exp2f(sm[w][row] - base);
      sum = __builtin_fmaf(sl[w][row], fw, sum);
      const f32x4 x = *reinterpret_cast<const f32x4*>(&so[w][row][4 * i]);
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = __builtin_fmaf(x[u], fw, v[u]);
    }
    if (parts == 1) {
      finish(row, i, v, top, sum);
    } else {
      put_quad(mine, words, e, v);
      if (i == 0) put_quad(mine, words, kRows * quads + row, f32x4{top, sum, 0.0f, 0.0f});
    }
  }
  if (parts == 1 || !last_to_arrive(f.arrived + group, parts)) return;
  const float* all = f.part + group * f.splits * words * 4;
  // Every part's maximum and sum; what each part weighs, and the row's own.
  float* tops = &so[0][0][0];            // [kRows][kMaxParts]
  float* sums = tops + kRows * kMaxParts;
  static_assert(sizeof(so) >= 2 * kRows * kMaxParts * sizeof(float), "the parts' statistics in LDS");
  for (int e = threadIdx.x; e < valid * parts; e += kAttnThreads) {
    const f32x4 x = get_quad(all + (int64_t)(e / valid) * words * 4, words, kRows * quads + e % valid);
    tops[e % valid * kMaxParts + e / valid] = x[0];
    sums[e % valid * kMaxParts + e / valid] = x[1];
  }
  __syncthreads();
  {
    const int row = threadIdx.x / 16, j = threadIdx.x % 16;   // sixteen lanes a row
    float top = -__builtin_inff();
    if (row < valid)
      for (int i = j; i < parts; i += 16) top = fmaxf(top, tops[row * kMaxParts + i]);
#pragma unroll
    for (int x = 8; x; x >>= 1) top = fmaxf(top, __shfl_xor(top, x, 16));
    const float base = top == -__builtin_inff() ? 0.0f : top;
    float sum = 0.0f;
    if (row < valid)
      for (int i = j; i < parts; i += 16) {
        const float w = __builtin_amdgcn_exp2f(tops[row * kMaxParts + i] - base);
        tops[row * kMaxParts + i] = w;
        sum = __builtin_fmaf(sums[row * kMaxParts + i], w, sum);
      }
#pragma unroll
    for (int x = 8; x; x >>= 1) sum += __shfl_xor(sum, x, 16);
    if (j == 0) {
      sm[0][row] = top;
      sl[0][row] = sum;
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < valid * quads; e += kAttnThreads) {
    const int row = e / quads;
    f32x4 v = {};
    for (int p = 0; p < parts; p += 8) {   // eight parts' loads in flight, added in order
      f32x4 x[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) x[u] = get_quad(all + (int64_t)min(p + u, parts - 1) * words * 4, words, e);
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float w = p + u < parts ? tops[row * kMaxParts + p + u] : 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = p + u < parts ? __builtin_fmaf(x[u][i], w, v[i]) : v[i];
      }
    }
    finish(row, e % quads, v, sm[0][row], sl[0][row]);
  }
}

// How the positions are cut. A workgroup's way into its stream and out of it costs
// some microseconds, so a sequence is cut only where the rows' tiles alone leave
// the chip empty: into 512 workgroups together, or, in pieces of 1280 positions
// or more, into 2048 (they even out what the lengths do not). Measured, in us,
// for 512 / 1024 / 2048: 64 rows of 1024, 8 heads of 128: 54 / 72 / 68 (8-bit 32
// / 41 / 44); 8 rows of 2000, 20 heads of 64: 17.7 / 18.5 / 19.9; 6 rows of 12000
// to 50001, 8 heads of 128, 8-bit: 95 / 94 / 87.
FewArgs few_args(const AttnArgs& a) {
  FewArgs f{};
  f.a = a;
  f.tiles = (int)(((int64_t)a.max_new * a.shared + kRows - 1) / kRows);
  const int64_t cap = (int64_t)a.c.max_pages << a.c.page_shift, groups = (int64_t)f.tiles * a.c.n_heads * a.c.n_seqs;
  const int64_t coarse = std::max<int64_t>(512 / groups, 1), fine = std::max<int64_t>(2048 / groups, 1);
  int64_t chunk = std::min(cap / coarse, std::max<int64_t>(1280, cap / fine)) + 255;
  chunk = std::max(chunk, (cap + kMaxParts - 1) / kMaxParts + 255) / 256 * 256;
  f.chunk = (int)std::min<int64_t>(std::max<int64_t>(chunk, 256), (int64_t)kMaxPages << a.c.page_shift);
  f.splits = (int)std::max<int64_t>((cap + f.chunk - 1) / f.chunk, 1);
  return f;
}

template <int DH, bool Q8, bool FULL, int KEYS>
hipError_t few(const FewArgs& f, hipStream_t s) {
  hipLaunchKernelGGL((k_attn_few<DH, Q8, FULL, KEYS>), dim3((unsigned)((int64_t)f.tiles * f.splits * f.a.c.n_heads), f.a.c.n_seqs),
                     dim3(kAttnThreads), 0, s, f);
  return hipGetLastError();
}
template <int DH, int BKEYS, int QKEYS>
hipError_t few(const FewArgs& f, hipStream_t s) {
  const bool full = f.a.c.dim == DH;
  if (f.a.c.store == C4S_KV_Q8) return full ? few<DH, true, true, QKEYS>(f, s) : few<DH, true, false, QKEYS>(f, s);
  return full ? few<DH, false, true, BKEYS>(f, s) : few<DH, false, false, BKEYS>(f, s);
}

// ---- many rows ----------------------------------------------------------------------------
//
// Prompts: a workgroup has 16 NB W rows of one sequence and key head, 16 NB a
// wave, and goes through the positions in blocks of 64, which all W waves
// share: a block's keys and values are loaded (codes converted, once for all
// rows) into registers while the block before it is worked on, and written to
// the other of two buffers in LDS, with one barrier a block. The rows of both
// buffers are permuted in 16-byte pieces so that the fragment reads of sixteen
// lanes that LDS serves together fall into different banks. Blocks behind a
// wave's last row are skipped by it, masks are applied only where a block
// holds the limit of some row, and the tiles with the most positions start
// first, those of up to 64 sequences together (of one after the other: 8 of 2048,
// 20 heads of 64, 169 us for 152; 4 of 2000, 10 query heads on 5 of 256, 195 for 172).
//
// What bounds it (20 heads of 64, 12 prompts of 500 to 2100): the VALU, 63 % busy;
// the matrix engine is 22 %, LDS 35 % (a tenth of it bank conflicts). Heads of 256
// have two waves a SIMD, which wait 60 % of the time, with LDS at 35, VALU at 29 and
// matrix engine at 23 %; the compiler spills 18 registers of theirs, and 10 of those of
// 8-bit heads of 64.
//
// Weights for bf16 values enter the second product rounded to bf16 once:
// independent roundings of 2^-9 at most, which leave 1.15 to 1.4 times the error of
// the output's own rounding (the largest weight is often 1, which has none). As
// pairs, as with few rows, they would add nothing to it, for half as many matrix instructions
// again and the VALU's splitting (pairs / once, us: 8 of 2048, 20 heads of 64 194 / 157;
// 2 of 4096, 32 query heads on 8 of 128 441 / 338; 4 of 2000, 5 heads of 256 125 / 105;
// 64 of 20 to 100 21.5 / 19).
// Weights for codes have the values' scales in them, none is exact, and the error
// would come to 1.5 times: those enter as pairs (8 prompts of 2048, 20 heads of 64:
// 224 us for 185, 1.0 times). The weights' sum is taken before the rounding, in fp32
// (from the matrix engine, of the rounded weights, it would be cheaper and lse off by 3e-4).
constexpr int kBlock = 64;         // positions
constexpr int kSegment = 16384;    // positions whose pages LDS holds at a time
constexpr float kSlack = 8.0f;     // weights stay below 2^kSlack: rows are rescaled only when that would not hold

struct ManyArgs {
  AttnArgs a;
  int tiles, together;   // sequences whose tiles start together
};

// Where row r of a block of keys (NP pieces a row) keeps piece p, and row r of
// one of values (eight pieces). LDS serves lanes 0-3, 12-15, 20-23 and 24-27 (and
// so on) together: those read rows 16 apart (keys) or next to each other
// (values), and in two lane groups' pieces.
template <int NP>
__device__ __forceinline__ int key_piece(int r, int p) {
  const int f = NP == 8 ? ((r >> 1) & 1) | ((r >> 4) & 3) << 1 : (r & 3) | ((r >> 4) & 3) << 2;
  return (r * NP + (p ^ f)) * 16;
}
__device__ __forceinline__ int value_piece(int r, int p) {
  return (r * 8 + (p ^ (((r >> 1) & 1) << 1 | ((r >> 2) & 1) | ((r >> 3) & 1) << 2))) * 16;
}

template <int DH, bool Q8, int NB, int W, int OCC>
__global__ __launch_bounds__(64 * W, OCC) void k_attn_many(ManyArgs f) {
  constexpr int kSteps = DH / 32, kTiles = DH / 16, kNP = DH / 8;   // kNP: pieces of a key
  constexpr int kThreads = 64 * W, kPieces = kBlock * DH / (Q8 ? 16 : 8);      // of a block's keys, and of its values
  constexpr int kLoads = kPieces < kThreads ? 1 : kPieces / kThreads;               // a thread's
  constexpr int kStagers = kPieces < kThreads ? kPieces : kThreads;                 // threads that have some
  constexpr int kBuf = 2 * kBlock * DH * 2;
  __shared__ __align__(16) char lds[2][kBuf];
  __shared__ __align__(16) float scales[2][Q8 ? 2 * kBlock : 4];    // [buffer][keys', values']
  __shared__ int32_t pages[kSegment / 16];
  // Values that are not finite where only some of a block's rows see them: by dim (codes: for all dims), the
  // first position of one. They enter the products as zeros, and rows that end behind it become NaN. (What an
  // earlier block left here did that already to the rows it is for.)
  __shared__ int bad[Q8 ? 1 : DH];
  __shared__ int odd[2][W];   // whether a wave staged such values
  __shared__ int gaps[W];     // whether a wave found a page of the segment missing
  const AttnArgs& a = f.a;
  const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64, c = lane % 16, g = lane / 16;
  const int dim = a.c.dim, pairs = a.c.n_heads * f.together, tile = f.tiles - 1 - blockIdx.x / pairs;
  const int head = blockIdx.x % pairs % a.c.n_heads, seq = blockIdx.y * f.together + blockIdx.x % pairs / a.c.n_heads;
  if (seq >= a.c.n_seqs) return;
  const Seq sq(a, seq);
  const int n_all = sq.n_new * a.shared, r0 = tile * 16 * NB * W;
  if (r0 >= n_all) return;
  const int fst = sq.fst, shift = a.c.page_shift, ps = 1 << shift;
  auto token_of = [&](int r) { return a.shared == 1 ? r : r / a.shared; };
  // This wave's rows; a lane has row 16 b + c of each block b.
  const int w0 = r0 + 16 * NB * wave;
  const bool any_rows = w0 < n_all;
  int lim[NB], least = 0, most = 0;   // least, most: of the wave's first and last row
  const uint16_t* qp[NB];
  uint16_t* op[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const int r = min(w0 + 16 * b + c, n_all - 1), token = token_of(r), qh = head * a.shared + r - token * a.shared;
    lim[b] = min(sq.past + token + 1, sq.cap);
    qp[b] = a.q + (int64_t)(sq.row0 + token) * a.ldq + qh * dim;
    op[b] = a.out + (int64_t)(sq.row0 + token) * a.ld_out + qh * dim;
  }
  if (any_rows) {
    least = min(sq.past + token_of(w0) + 1, sq.cap);
    most = min(sq.past + token_of(min(w0 + 16 * NB - 1, n_all - 1)) + 1, sq.cap);
  }
  const int kend = min(sq.past + token_of(min(r0 + 16 * NB * W - 1, n_all - 1)) + 1, sq.cap);   // the workgroup's last

  const int first_lim = min(sq.past + token_of(r0) + 1, sq.cap);                              // ... and its first

  // Scores become powers of two's exponents by one multiplication with a positive factor: a negative scale
  // turns q's signs, and none at all is so small that the weights are equal.
  const uint32_t turn = a.scale < 0.0f ? 0x80008000u : 0u;
  const float c2 = fmaxf(fabsf(a.scale) * kLog2e, 0x1p-100f);
  uint4 q[NB][kSteps];
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const uint4 w = 32 * s + 8 * g < dim ? *reinterpret_cast<const uint4*>(qp[b] + 32 * s + 8 * g) : make_uint4(0, 0, 0, 0);
      q[b][s] = make_uint4(w.x ^ turn, w.y ^ turn, w.z ^ turn, w.w ^ turn);
    }

  constexpr int kSize = Q8 ? 1 : 2;
  const uint32_t head_bytes = (uint32_t)(dim * kSize) << shift, page_bytes = head_bytes * (uint32_t)a.c.n_heads;
  const char* kbase = static_cast<const char*>(a.c.k) + (uint64_t)head_bytes * head;
  const char* vbase = static_cast<const char*>(a.c.v) + (uint64_t)head_bytes * head;
  const int32_t* table = a.c.table + (int64_t)seq * a.c.table_ld;
  float m[NB];   // what the weights are relative to (as exponents of two), within kSlack of the maximum seen
  float l[NB];   // a lane's part of the weights' sum
  f32x4 o[NB][kTiles] = {};
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    m[b] = -__builtin_inff();
    l[b] = 0.0f;
  }

  for (int i = tid; i < (Q8 ? 1 : DH); i += kThreads) bad[i] = INT32_MAX;
  // (From fst < kend on, a segment's first block begins before its end: its table holds every block's pages.)
  for (int seg = fst & ~(kSegment - 1); fst < kend && seg < kend; seg += kSegment) {
    const int begin = max(seg, fst & ~(kBlock - 1)), end = min(seg + kSegment, kend);
    if (seg > fst) __syncthreads();   // the segment before has been read
    bool missing = false;             // whether a page of the segment is not there
    for (int i = tid; i < (((end - seg + kBlock - 1) & ~(kBlock - 1)) + ps - 1) >> shift; i += kThreads) {   // through the last block
      const int at = (seg >> shift) + i;
      const int p = at < a.c.max_pages ? table[at] : -1;
      pages[i] = p < a.c.n_pages ? p : -1;
      missing |= (p < 0 || p >= a.c.n_pages) && (i + 1) * ps + seg > fst && i * ps + seg < end;
    }
    missing = __any(missing);
    if (lane == 0) gaps[wave] = missing;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; ++w) missing |= gaps[w] != 0;
    uint4 kst[kLoads], vst[kLoads];
    float sst = 0.0f;
    // A thread's pieces of a block: of the keys in order; of the values in the order in which a page has them.
    // A block begins at a multiple of 64, so that of a piece's place in its page and in the table only what
    // the block adds changes.
    constexpr int kKP = Q8 ? DH / 16 : DH / 8, kPer = Q8 ? 16 : 8;   // a key's pieces; dims or positions a piece
    const int row_shift = min(shift, 6) - (Q8 ? 4 : 3);              // log2 of the pieces a page's row has in a block
    auto key_of = [&](int i) { return (tid + kThreads * i) / kKP; };
    auto dim_of = [&](int i) { return ((tid + kThreads * i) >> row_shift) % DH; };   // of a piece of values, and which of its row
    auto piece_of = [&](int i) {
      const int at = tid + kThreads * i;
      return (at >> row_shift) / DH << row_shift | (at & ((1 << row_shift) - 1));
    };
    auto page_at = [&](int t, int in) { return (uint64_t)(uint32_t)max(pages[((t - seg) >> shift) + (in >> shift)], 0); };   // what has no page is dropped
    auto load = [&](int t) {
      const uint32_t key_add = (uint32_t)((t & (ps - 1)) * dim * kSize), value_add = (uint32_t)((t & (ps - 1)) * kSize);
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        if (kStagers < kThreads && tid >= kStagers) break;
        const int d = tid % kKP * kPer;   // the threads are a multiple of a key's pieces
        kst[i] = make_uint4(0, 0, 0, 0);
        if (d < dim)
          kst[i] = *reinterpret_cast<const uint4*>(kbase + key_add + page_at(t, key_of(i)) * page_bytes + (uint32_t)(((key_of(i) & (ps - 1)) * dim + d) * kSize));
        const int pos = piece_of(i) * kPer;
        vst[i] = *reinterpret_cast<const uint4*>(vbase + value_add + page_at(t, pos) * page_bytes + (uint32_t)(((min(dim_of(i), dim - 1) << shift) + (pos & (ps - 1))) * kSize));
      }
      if constexpr (Q8) {
        if (tid < 2 * kBlock) {
          const int pos = t + tid % kBlock;
          sst = (tid < kBlock ? a.c.k_scale : a.c.v_scale)[(page_at(t, tid % kBlock) * a.c.n_heads + head << shift) + (pos & (ps - 1))];
        }
      }
    };
    auto edge_of = [&](int t) { return t < fst || t + kBlock > first_lim || missing; };
    auto stage = [&](int t, int buf) {
      char* kl = lds[buf];
      char* vl = kl + kBlock * DH * 2;
      // What is not there or not for any row may hold anything: zeros (codes: their scales).
      int strange = 0;
      const bool edge = edge_of(t);
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        if (kStagers < kThreads && tid >= kStagers) break;
        const int vd = dim_of(i), piece = piece_of(i);
        if constexpr (Q8) {
          *reinterpret_cast<uint4*>(kl + key_piece<kNP>(key_of(i), tid % kKP * 2)) = codes(make_uint2(kst[i].x, kst[i].y));
          *reinterpret_cast<uint4*>(kl + key_piece<kNP>(key_of(i), tid % kKP * 2 + 1)) = codes(make_uint2(kst[i].z, kst[i].w));
          *reinterpret_cast<uint4*>(vl + value_piece(vd, 2 * piece)) = codes(make_uint2(vst[i].x, vst[i].y));
          *reinterpret_cast<uint4*>(vl + value_piece(vd, 2 * piece + 1)) = codes(make_uint2(vst[i].z, vst[i].w));
        } else {
          *reinterpret_cast<uint4*>(kl + key_piece<kNP>(key_of(i), tid % kKP)) = kst[i];
          if (edge) {
            const int pos = t + 8 * piece;
            if (t < fst || t + kBlock > kend || missing)
              vst[i] = keep(vst[i], 0, fst - pos, pages[(pos - seg) >> shift] >= 0 ? kend - pos : 0);
            if (any_odd(vst[i])) {
              strange = 1;
              uint32_t w[4] = {vst[i].x, vst[i].y, vst[i].z, vst[i].w}, was;
#pragma unroll
              for (int j = 3; j >= 0; --j) {
                part_odd(w[j], was);
                if (was) atomicMin(&bad[vd], pos + 2 * j + (was & 0xFFFFu ? 0 : 1));
              }
              vst[i] = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
          *reinterpret_cast<uint4*>(vl + value_piece(vd, piece)) = vst[i];
        }
      }
      if constexpr (Q8) {
        if (tid < 2 * kBlock) {
          const int pos = t + tid % kBlock;
          if (edge && (pos < fst || pos >= kend || pages[(pos - seg) >> shift] < 0)) sst = 0.0f;
          if (edge && tid >= kBlock && !(sst - sst == 0.0f)) {
            strange = 1;
            sst = 0.0f;
            atomicMin(&bad[0], pos);
          }
          scales[buf][tid] = sst;
        }
      }
      const bool mark = __any(strange);
      if (lane == 0) odd[buf][wave] = mark;
    };
    load(begin);
    stage(begin, 0);
    if (begin + kBlock < end) load(begin + kBlock);
    int buf = 0;
    for (int t = begin; t < end; t += kBlock, buf ^= 1) {
      __syncthreads();   // this block is there, and the other buffer has been read
      if (t + kBlock < end) {
        stage(t + kBlock, buf ^ 1);
        if (t + 2 * kBlock < end) load(t + 2 * kBlock);
      }
      if (t >= most) continue;   // no row of this wave sees it
      const char* kl = lds[buf];
      const char* vl = kl + kBlock * DH * 2;
      f32x4 s[NB][4] = {};
#pragma unroll
      for (int tt = 0; tt < 4; ++tt)
#pragma unroll
        for (int st = 0; st < kSteps; ++st) {
          const uint4 w = *reinterpret_cast<const uint4*>(kl + key_piece<kNP>(16 * (c / 4) + 4 * tt + c % 4, 4 * st + g));
#pragma unroll
          for (int b = 0; b < NB; ++b) s[b][tt] = mfma(w, q[b][st], s[b][tt]);
        }
      const int vt = t + 16 * g;   // a lane's 16 positions
      if constexpr (Q8) {
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) {
          const f32x4 ks = *reinterpret_cast<const f32x4*>(&scales[buf][16 * g + 4 * tt]);
#pragma unroll
          for (int b = 0; b < NB; ++b) s[b][tt] *= ks;
        }
      }
      if (t + kBlock > least || missing) {
        const bool there = pages[(vt - seg) >> shift] >= 0;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const int to = there ? lim[b] - vt : 0;
#pragma unroll
          for (int j = 0; j < 16; ++j) s[b][j / 4][j % 4] = j < to ? s[b][j / 4][j % 4] : -__builtin_inff();
        }
      }
      if (t < fst) {
        const int from = fst - vt;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int j = 0; j < 16; ++j) s[b][j / 4][j % 4] = j < from ? -__builtin_inff() : s[b][j / 4][j % 4];
      }
      auto value = [&](int d, int st) { return *reinterpret_cast<const uint4*>(vl + value_piece(16 * d + c, 2 * g + st)); };
      constexpr bool kAhead = DH == 64;   // two dim tiles' values asked for before the weights, the others' before the products
      uint4 va[kAhead ? 4 : 1];
      if constexpr (kAhead) {
#pragma unroll
        for (int i = 0; i < 4; ++i) va[i] = value(i / 2, i % 2);
        __builtin_amdgcn_sched_barrier(0);
      }
      uint32_t p[NB][8], rest[NB][Q8 ? 8 : 1];
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        float top = fmaxf(s[b][0][0], s[b][0][1]);
#pragma unroll
        for (int j = 2; j < 16; ++j) top = fmaxf(top, s[b][j / 4][j % 4]);
        if (__any(top * c2 > m[b] + kSlack)) {   // seldom, after a row's first block
          top = fmaxf(max4(top) * c2, m[b]);
          const float old = __builtin_amdgcn_exp2f(m[b] - (top == -__builtin_inff() ? 0.0f : top));
          l[b] *= old;
#pragma unroll
          for (int d = 0; d < kTiles; ++d) o[b][d] *= old;
          m[b] = top;
        }
        const float base = m[b] == -__builtin_inff() ? 0.0f : m[b];   // nothing seen yet
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
          float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][j / 4][j % 4], c2, -base));
          float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][j / 4][j % 4 + 1], c2, -base));
          l[b] += x + y;
          if constexpr (Q8) {
            const f32x2 vs = *reinterpret_cast<const f32x2*>(&scales[buf][kBlock + 16 * g + j]);
            x *= vs[0];
            y *= vs[1];
          }
          p[b][j / 2] = pack(x, y);
          if constexpr (Q8) rest[b][j / 2] = pack(x - low(p[b][j / 2]), y - high(p[b][j / 2]));
        }
      }
      auto quad = [](const uint32_t* w) { return make_uint4(w[0], w[1], w[2], w[3]); };
      auto add = [&](f32x4& to, uint4 v, int b, int st) {
        to = mfma(v, quad(p[b] + 4 * st), to);
        if constexpr (Q8) to = mfma(v, quad(rest[b] + 4 * st), to);
      };
      if constexpr (kAhead) {
#pragma unroll
        for (int b = 0; b < NB; ++b) asm volatile("" : "+v"(l[b]));   // summed here: the weights' registers are free for values
        uint4 vb[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) vb[i] = value(2 + i / 2, i % 2);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int st = 0; st < 2; ++st)
#pragma unroll
          for (int d = 0; d < 2; ++d)
#pragma unroll
            for (int b = 0; b < NB; ++b) add(o[b][d], va[2 * d + st], b, st);
#pragma unroll
        for (int st = 0; st < 2; ++st)
#pragma unroll
          for (int d = 0; d < 2; ++d)
#pragma unroll
            for (int b = 0; b < NB; ++b) add(o[b][2 + d], vb[2 * d + st], b, st);
      } else {
#pragma unroll
        for (int d = 0; d < kTiles; ++d) {
          if (16 * d >= dim) break;
#pragma unroll
          for (int st = 0; st < 2; ++st) {
            const uint4 v = *reinterpret_cast<const uint4*>(vl + value_piece(16 * d + c, 2 * g + st));
#pragma unroll
            for (int b = 0; b < NB; ++b) add(o[b][d], v, b, st);
          }
        }
      }
      int strange = 0;
      if (!kAhead || edge_of(t)) {
#pragma unroll
        for (int w = 0; w < W; ++w) strange |= odd[buf][w];
      }
      if (strange) {
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int d = 0; d < kTiles; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (bad[Q8 ? 0 : 16 * d + 4 * g + i] < lim[b]) o[b][d][i] = __builtin_nanf("");
      }
    }
  }
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const float sum = sum4(l[b]);
    const int r = w0 + 16 * b + c;
    if (r >= n_all) continue;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int d = 0; d < kTiles; ++d) {
      if (16 * d >= dim) break;
      const f32x4 v = o[b][d] * inv;
      *reinterpret_cast<uint2*>(op[b] + 16 * d + 4 * g) = make_uint2(pack(v[0], v[1]), pack(v[2], v[3]));
    }
    if (a.lse && g == 0)
      a.lse[(int64_t)(sq.row0 + token_of(r)) * a.n_heads + head * a.shared + r - token_of(r) * a.shared] = sum == 0.0f ? -__builtin_inff() : (m[b] + log2f(sum)) * kLn2;
  }
}

template <int DH, bool Q8, int NB, int W, int OCC>
hipError_t many(const AttnArgs& a, hipStream_t s) {
  const int tiles = (int)(((int64_t)a.max_new * a.shared + 16 * NB * W - 1) / (16 * NB * W));
  // 64 sequences, or what the grid has room for (2^32 threads in a dimension)
  const int64_t room = (int64_t)(UINT32_MAX / (64 * W)) / ((int64_t)tiles * a.c.n_heads);
  const int together = (int)std::min<int64_t>(std::min(a.c.n_seqs, 64), std::max<int64_t>(room, 1));
  const ManyArgs f{a, tiles, together};
  hipLaunchKernelGGL((k_attn_many<DH, Q8, NB, W, OCC>), dim3((unsigned)((int64_t)f.tiles * a.c.n_heads * together), (a.c.n_seqs + together - 1) / together),
                     dim3(64 * W), 0, s, f);
  return hipGetLastError();
}

// Few rows' tiles re-read the positions but share them out over the chip: they win while they are few, and where
// the other kernel would leave most rows of a workgroup empty. Few / many rows' kernel, us, by tiles: bf16, 20 heads
// of 64: 1 of 500 rows, 640, 9.2 / 11.8; 4 of 128 over 4000, 640, 72 / 66; 2 of 300, 760, 8.1 / 8.2; 4 of 300 over 500,
// 1520, 31 / 18; 8 key heads of 128 with 4 query heads each: 1 of 300, 600, 15.5 / 18.9; 2 of 200 over 1000, 800, 70 /
// 50. 8-bit codes are converted for each block of the many rows' kernel by all its waves: 20 heads of 64: 4 of 128 over
// 1000, 640, 21 / 30; 2 of 600, 1520, 17.9 / 18.9; 4 of 300 over 500, 1520, 27 / 24; 64 of 48 and of 64 over 300,
// three and four tiles a sequence, 35 / 39 and 45 / 42; 8 heads of 128: 2 of 200 over 1000, 800, 43 / 65; 2 of 400 over 400, 1600, 48 / 48; 5 heads of 256: 4
// of 200 over 200, 500, 30 / 29; 4 of 500 over 500, 1260, 107 / 59.
bool many_pays(const AttnArgs& a) {
  const int64_t tiles = ((int64_t)a.max_new * a.shared + kRows - 1) / kRows, all = tiles * a.c.n_heads * a.c.n_seqs;
  if (a.c.store == C4S_KV_Q8 && a.c.dim <= 128) return tiles > 3 && all > 1500;
  return tiles > 1 && all > 700;
}

}  // namespace

LayerSpace attn_space(const AttnArgs& a) {
  if (many_pays(a)) return {};
  const FewArgs f = few_args(a);
  if (f.splits == 1) return {};
  // more threads than a grid has room for in its first dimension: more counters than there are, which the caller refuses
  if ((int64_t)f.tiles * f.splits * a.c.n_heads > (int64_t)(UINT32_MAX / kAttnThreads)) return {INT64_MAX / 4, 1};
  const int64_t groups = (int64_t)f.tiles * a.c.n_heads * a.c.n_seqs;
  return {groups, groups * f.splits * kRows * (a.c.dim + 4)};
}

hipError_t launch_attn(const AttnArgs& a, uint32_t* counters, float* space, hipStream_t s) {
  if (many_pays(a)) {
    if (a.c.dim <= 64) return a.c.store == C4S_KV_Q8 ? many<64, true, 1, 8, 4>(a, s) : many<64, false, 1, 8, 4>(a, s);
    if (a.c.dim <= 128) return a.c.store == C4S_KV_Q8 ? many<128, true, 2, 8, 2>(a, s) : many<128, false, 2, 8, 2>(a, s);
    return a.c.store == C4S_KV_Q8 ? many<256, true, 1, 8, 2>(a, s) : many<256, false, 1, 8, 2>(a, s);
  }
  FewArgs f = few_args(a);
  f.arrived = counters;
  f.part = space;
  if (a.c.dim <= 64) return few<64, 32, 32>(f, s);
  if (a.c.dim <= 128) return few<128, 32, 64>(f, s);
  return few<256, 32, 32>(f, s);
}

}  // namespace c4s
