// The paged key-value cache: rows written as bf16 or as 8- or 4-bit codes, and
// read back (include/c4s_layers.h has the layout).
//
// Both kernels take tiles of packed rows of one head, four lanes a row (a read in large
// tiles eight, with two rows each). Keys keep
// their order: pieces of eight dims go to and from the page as they are. Values
// lie in the page with their positions next to each other, so a tile of them
// passes through LDS. Four rows of a tile that are positions 4 i .. 4 i + 3 of a
// page (all but the ends of a prompt) are stored and loaded together, 16 such
// groups of a dim next to each other; others (a step's single tokens) one by one.
// The heads of a tile follow each other in the grid: a row's 128 bytes a head
// are then read and written next to each other in time.
//
// Memory bounds both for prompts, and both move more than they need. 24 prompts of
// 70 to 1500 tokens, 20 heads of 64, 8-bit, calls back to back: the read needs 179 MB
// (62 of codes and scales, 117 of rows) and takes 37 us, 4.8 TB/s, in which 93 and
// 117 MB pass; the write needs 148 MB (96 of rows, 51 of codes and scales) and takes
// 51 us, 2.9 TB/s, in which 97 and 65 MB pass. What the write adds are the
// lines of pages that a tile's ends leave half full; the VALU, which computes the
// codes, is busy half of the time, and which of the two costs more is not known.
// In 4 bits (18829 rows like those, from memory / from the last-level cache) the write's 121 MB
// take 39 / 30 us, the read's as many 25 / 25, 4.9 TB/s; 64 rows 4.1 and 4.6.

#include <hip/hip_runtime.h>

#include <type_traits>

#include "c4s_layers.hpp"

namespace c4s {
namespace {

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
    while (hi - lo > 1) {        // eight parts a step: each step is a wait for memory
      const int step = (hi - lo + 7) / 8;
      int behind = 0;
#pragma unroll
      for (int j = 1; j < 8; ++j) behind += (lo + j * step < hi) & (off[min(lo + j * step, hi - 1)] <= r);
      lo += behind * step;
      hi = min(lo + step, hi);
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

typedef uint32_t Piece __attribute__((ext_vector_type(4), aligned(8)));   // eight bf16
typedef uint32_t Codes __attribute__((ext_vector_type(2)));               // eight codes
typedef uint16_t Halves __attribute__((ext_vector_type(2)));
typedef __bf16 Pair __attribute__((ext_vector_type(2)));                  // rounds to nearest even

__device__ __forceinline__ float from_bf16(uint32_t h) { return __uint_as_float(h << 16); }

// Over the four lanes of a row (quad_perm).
__device__ __forceinline__ uint32_t max4(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, v, 0xB1, 0xF, 0xF, true));
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, v, 0x4E, 0xF, 0xF, true));
}

// Where a tile's rows lie, and which of them go together: `lead` the rows that
// begin a group of four, `single` those in none.
template <int TILE>
struct Tile {
  Place at[TILE];
  uint8_t lead[TILE / 4], single[TILE];
  int n_lead, n_single;

  __device__ __forceinline__ void find(const KvArgs& c, const KvRowsArgs& rows) {
    if (threadIdx.x < 64) {   // one wave: a lane a row
      const int r = threadIdx.x;
      Place p{-1, 0};
      if (r < TILE) {
        p = place_of(c, rows.lens, rows.off, rows.n_rows, blockIdx.x / c.n_heads * TILE + r);
        at[r] = p;
      }
      const int page = (int)p.page;
      const bool row = page >= 0;
      // rows whose next one follows them in their page; four in line from a multiple of four on go together
      const uint64_t next = __ballot(row & (__shfl_down(page, 1) == page) & (__shfl_down(p.at, 1) == p.at + 1));
      const uint64_t lm = __ballot(row & !(p.at & 3)) & next & next >> 1 & next >> 2;
      const uint64_t sm = __ballot(row) & ~(lm | lm << 1 | lm << 2 | lm << 3), below = (1ull << r) - 1;
      if (lm >> r & 1) lead[__popcll(lm & below)] = (uint8_t)r;
      if (sm >> r & 1) single[__popcll(sm & below)] = (uint8_t)r;
      if (r == 0) {
        n_lead = __popcll(lm);
        n_single = __popcll(sm);
      }
    }
    __syncthreads();
  }
};

// The bytes of four words exchanged, as a 4 x 4 matrix is transposed.
__device__ __forceinline__ void transpose_bytes(uint32_t (&x)[4]) {
  const uint32_t lo01 = __builtin_amdgcn_perm(x[1], x[0], 0x05010400), hi01 = __builtin_amdgcn_perm(x[1], x[0], 0x07030602);
  const uint32_t lo23 = __builtin_amdgcn_perm(x[3], x[2], 0x05010400), hi23 = __builtin_amdgcn_perm(x[3], x[2], 0x07030602);
  x[0] = __builtin_amdgcn_perm(lo23, lo01, 0x05040100);
  x[1] = __builtin_amdgcn_perm(lo23, lo01, 0x07060302);
  x[2] = __builtin_amdgcn_perm(hi23, hi01, 0x05040100);
  x[3] = __builtin_amdgcn_perm(hi23, hi01, 0x07060302);
}
// The halves of (x, y) as (low halves, high halves).
__device__ __forceinline__ void swap_halves(uint32_t& x, uint32_t& y) {
  const uint32_t lo = __builtin_amdgcn_perm(y, x, 0x05040100);
  y = __builtin_amdgcn_perm(y, x, 0x07060302);
  x = lo;
}

// Eight values as codes of four bits, and back: a block's scale is 2^(e - 127), e its byte, which is a float's exponent.
__device__ __forceinline__ float scale4(uint32_t e) { return __uint_as_float(e << 23); }
__device__ __forceinline__ uint32_t codes4(const Piece& w, float scale) {
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(Pair, (uint32_t)w[0]), scale, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(Pair, (uint32_t)w[1]), scale, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(Pair, (uint32_t)w[2]), scale, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(Pair, (uint32_t)w[3]), scale, 3);
}
__device__ __forceinline__ Piece values4(uint32_t c, float scale) {
  return Piece{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 0)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 1)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 2)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 3))};
}

// A tile of values in LDS, a row as it is outside the cache. An odd row length puts
// the words that a wave moves between it and the pages in banks of their own.
// (4-bit codes move as 8-bit ones of half as many dims: a byte is a pair of dims.)
template <int STORE, int PIECES, int TILE>
struct Values {
  static constexpr bool Q8 = STORE != C4S_KV_BF16;
  static constexpr int kThreads = 4 * TILE, kGroups = TILE / 4, kDims = STORE == C4S_KV_Q4 ? 8 : (Q8 ? 4 : 2);   // of a word
  uint32_t words[TILE][PIECES * 32 / kDims + 1];

  __device__ __forceinline__ uint32_t* piece(int row, int d) { return &words[row][d / kDims]; }

  // To (TO_PAGES) or from the pages' rows of positions; v0: where a place's position
  // of dim 0 lies. Then words of four dims (Q8) or two for four positions at once.
  template <bool TO_PAGES, class V0>
  __device__ __forceinline__ void move(const Tile<TILE>& tile, int dim, int shift, V0 v0) {
    if ((int)threadIdx.x % kGroups < tile.n_lead) {
      const int g = tile.lead[threadIdx.x % kGroups];
      uint8_t* at = v0(tile.at[g]);
#pragma unroll 2
      for (int w = threadIdx.x / kGroups; w * (Q8 ? 4 : 2) < dim; w += kThreads / kGroups) {
        uint32_t x[4];
        if (TO_PAGES) {
#pragma unroll
          for (int j = 0; j < 4; ++j) x[j] = words[g + j][w];
        }
        if (Q8) {
          uint8_t* p = at + ((uint32_t)(4 * w) << shift);
          if (!TO_PAGES) {
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = *reinterpret_cast<const uint32_t*>(p + ((uint32_t)j << shift));
          }
          transpose_bytes(x);
          if (TO_PAGES) {
#pragma unroll
            for (int j = 0; j < 4; ++j) *reinterpret_cast<uint32_t*>(p + ((uint32_t)j << shift)) = x[j];
          }
        } else {
          uint2* p0 = reinterpret_cast<uint2*>(at + ((uint32_t)(4 * w) << shift));
          uint2* p1 = reinterpret_cast<uint2*>(at + ((uint32_t)(4 * w + 2) << shift));
          if (TO_PAGES) {
            swap_halves(x[0], x[1]);
            swap_halves(x[2], x[3]);
            *p0 = make_uint2(x[0], x[2]);
            *p1 = make_uint2(x[1], x[3]);
          } else {
            const uint2 a = *p0, b = *p1;
            x[0] = a.x, x[1] = b.x, x[2] = a.y, x[3] = b.y;
            swap_halves(x[0], x[1]);
            swap_halves(x[2], x[3]);
          }
        }
        if (!TO_PAGES) {
#pragma unroll
          for (int j = 0; j < 4; ++j) words[g + j][w] = x[j];
        }
      }
    }
    using T = std::conditional_t<Q8, uint8_t, uint16_t>;
    for (int i = threadIdx.x % TILE; i < tile.n_single; i += TILE) {
      const int g = tile.single[i];
      T* at = reinterpret_cast<T*>(v0(tile.at[g]));
      T* mine = reinterpret_cast<T*>(words[g]);
#pragma unroll 4
      for (int d = threadIdx.x / TILE; d < dim; d += kThreads / TILE) {
        if (TO_PAGES) at[(uint32_t)d << shift] = mine[d];
        else mine[d] = at[(uint32_t)d << shift];
      }
    }
  }
};

// PIECES: of eight dims that a lane has of a row, at most.
//
// A code is value / scale to nearest even. One correction of the product with the
// rounded reciprocal gives the rounded quotient (Markstein 1990) where nothing
// leaves the range; adding 1.5 * 2^23 then leaves the integer to nearest even in
// the sum's low bits. (With divisions the prompts above take 58 us for 52, a
// step's 64 rows 4.8 for 4.1.)
// In 4 bits a block's 32 dims are one piece of each of a row's four lanes. Its scale's
// exponent comes from the bits of the largest magnitude: 6 is 1.5 * 2^2, so adding 0x3F
// to the 7 bits of the mantissa carries into the exponent just above 1.5.
template <int STORE, int PIECES, int TILE>
__global__ __launch_bounds__(4 * TILE, 4) void k_kv_append(KvArgs c, KvRowsArgs rows) {
  constexpr bool Q8 = STORE == C4S_KV_Q8, Q4 = STORE == C4S_KV_Q4;
  __shared__ Tile<TILE> tile;
  __shared__ Values<STORE, PIECES, TILE> values;
  const int row = threadIdx.x / 4, l = threadIdx.x % 4, dim = c.dim, ps = 1 << c.page_shift;
  const int head = blockIdx.x % c.n_heads;
  const int64_t r = (int64_t)(blockIdx.x / c.n_heads) * TILE + row;
  Piece raw[2][PIECES];   // underway while the places are looked up
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const uint16_t* src = static_cast<const uint16_t*>(which ? rows.v : rows.k) + r * (which ? rows.ldv : rows.ldk) + head * dim;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int d = 32 * i + 8 * l;
      raw[which][i] = r < rows.n_rows && d < dim ? *reinterpret_cast<const Piece*>(src + d) : Piece{};
    }
  }
  tile.find(c, rows);
  const Place p = tile.at[row];
  const int64_t slot = (p.page * c.n_heads + head) * (int64_t)ps + p.at;   // (position, head) in the cache
#pragma unroll
  for (int which = 1; which >= 0; --which) {   // the values first: their stores wait for the other lanes
    if (Q8) {
      // |value| by its bits, which order as the numbers do, with NaN past infinity
      Halves top = {};
#pragma unroll
      for (int i = 0; i < PIECES; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) top = __builtin_elementwise_max(top, __builtin_bit_cast(Halves, raw[which][i][j] & 0x7FFF7FFFu));
      const uint32_t most = max4(max(top[0], top[1]));
      // a value that is not finite makes the scale NaN, and so the row
      const float scale = most < 0x7F80u ? from_bf16(most) / 127.0f : __builtin_nanf("");
      if (p.page >= 0 && l == 0) (which ? c.v_scale : c.k_scale)[slot] = scale;
      const float inv = 1.0f / scale;
      const bool in_range = scale > 0x1p-60f && scale < 0x1p60f;
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        uint32_t sum[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float v = __uint_as_float(j % 2 ? raw[which][i][j / 2] & 0xFFFF0000u : raw[which][i][j / 2] << 16);
          const float q = v * inv;
          sum[j] = __float_as_uint(fmaf(fmaf(-q, scale, v), inv, q) + 12582912.0f);
        }
        if (!in_range) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float v = __uint_as_float(j % 2 ? raw[which][i][j / 2] & 0xFFFF0000u : raw[which][i][j / 2] << 16);
            sum[j] = scale > 0.0f ? __float_as_uint(v / scale + 12582912.0f) : 0u;
          }
        }
#pragma unroll
        for (int j = 0; j < 2; ++j)
          raw[which][i][j] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(sum[4 * j + 3], sum[4 * j + 2], 0x0C0C0400),
                                                   __builtin_amdgcn_perm(sum[4 * j + 1], sum[4 * j], 0x0C0C0400), 0x05040100);
      }
    }
    if (Q4) {
      uint8_t* scales = reinterpret_cast<uint8_t*>(which ? c.v_scale : c.k_scale) + (p.page * c.n_heads + head) * (int64_t)(dim / 32) * ps + p.at;
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        Halves top = {};
#pragma unroll
        for (int j = 0; j < 4; ++j) top = __builtin_elementwise_max(top, __builtin_bit_cast(Halves, raw[which][i][j] & 0x7FFF7FFFu));
        const uint32_t most = max4(max(top[0], top[1]));
        const uint32_t e = most >= 0x7F80u ? 255u : (uint32_t)max((int)((most + 0x3Fu) >> 7) - 2, 0);
        raw[which][i][0] = codes4(raw[which][i], scale4(e));
        if (p.page >= 0 && l == i % 4 && 32 * i < dim) scales[(uint32_t)i << c.page_shift] = (uint8_t)e;
      }
    }
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int d = 32 * i + 8 * l;
      if (p.page < 0 || d >= dim) continue;
      if (which) {
#pragma unroll
        for (int j = 0; j < (Q4 ? 1 : (Q8 ? 2 : 4)); ++j) values.piece(row, d)[j] = raw[1][i][j];
      } else if (Q4) {
        *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(c.k) + (slot * dim + d) / 2) = raw[0][i][0];
      } else if (Q8) {
        *reinterpret_cast<Codes*>(static_cast<uint8_t*>(c.k) + slot * dim + d) = Codes{raw[0][i][0], raw[0][i][1]};
      } else {
        *reinterpret_cast<Piece*>(static_cast<uint16_t*>(c.k) + slot * dim + d) = raw[0][i];
      }
    }
  }
  __syncthreads();
  const int wide = Q4 ? dim / 2 : dim;   // of a page's rows of positions
  values.template move<true>(tile, wide, c.page_shift, [&](const Place& q) {
    return static_cast<uint8_t*>(c.v) + ((q.page * c.n_heads + head) * (int64_t)ps * wide + q.at) * (STORE == C4S_KV_BF16 ? 2 : 1);
  });
}

// Four lanes a row; in large tiles eight, with two rows each, so that a store is a whole line (with four, past the caches,
// 158 MB are written where 117 are needed: the prompts above 50 us for 42 from memory, in 4 bits 30 for 26).
template <int STORE, int PIECES, int TILE>
__global__ __launch_bounds__(4 * TILE, 4) void k_kv_read(KvArgs c, KvRowsArgs rows) {
  constexpr bool Q8 = STORE == C4S_KV_Q8, Q4 = STORE == C4S_KV_Q4;
  constexpr int kLanes = TILE == 64 ? 8 : 4, kRows = kLanes / 4, kPieces = PIECES / kRows;
  __shared__ Tile<TILE> tile;
  __shared__ Values<STORE, PIECES, TILE> values;
  tile.find(c, rows);
  const int l = threadIdx.x % kLanes, dim = c.dim, ps = 1 << c.page_shift;
  const int head = blockIdx.x % c.n_heads;
  const auto row_of = [&](int h) { return (int)threadIdx.x / kLanes + TILE / kRows * h; };
  float scale[2][kRows];
  uint32_t e[2][kRows][Q4 ? kPieces : 1];
  Piece raw[2][kRows][kPieces];   // without a page: zeros
  bool mine[kRows], has[kRows];
#pragma unroll
  for (int h = 0; h < kRows; ++h) {
    const Place p = tile.at[row_of(h)];
    const int64_t slot = (p.page * c.n_heads + head) * (int64_t)ps + p.at;
    // a row between two sequences' rows, or behind the last, is not the call's to write
    const int64_t r = (int64_t)(blockIdx.x / c.n_heads) * TILE + row_of(h);
    mine[h] = r < rows.n_rows && (!rows.off || (r >= rows.off[0] && r < rows.off[c.n_seqs]));
    has[h] = p.page >= 0;
    scale[0][h] = scale[1][h] = 1.0f;
    if (Q8 && p.page >= 0) {
      scale[0][h] = c.k_scale[slot];
      scale[1][h] = c.v_scale[slot];
    }
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int d = 8 * (kLanes * i + l);
      raw[0][h][i] = raw[1][h][i] = Piece{};
      if (p.page < 0 || d >= dim) continue;
      if (Q4) {
        const int64_t at = (p.page * c.n_heads + head) * (int64_t)(dim / 32) * ps + p.at + ((uint32_t)(d / 32) << c.page_shift);
        e[0][h][i] = reinterpret_cast<const uint8_t*>(c.k_scale)[at];
        e[1][h][i] = reinterpret_cast<const uint8_t*>(c.v_scale)[at];
        raw[0][h][i][0] = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(c.k) + (slot * dim + d) / 2);
      } else if (Q8) {
        const Codes w = *reinterpret_cast<const Codes*>(static_cast<const uint8_t*>(c.k) + slot * dim + d);
        raw[0][h][i] = Piece{w[0], w[1], 0, 0};
      } else {
        raw[0][h][i] = *reinterpret_cast<const Piece*>(static_cast<const uint16_t*>(c.k) + slot * dim + d);
      }
    }
  }
  const int wide = Q4 ? dim / 2 : dim;   // of a page's rows of positions
  values.template move<false>(tile, wide, c.page_shift, [&](const Place& q) {
    return static_cast<uint8_t*>(c.v) + ((q.page * c.n_heads + head) * (int64_t)ps * wide + q.at) * (STORE == C4S_KV_BF16 ? 2 : 1);
  });
  __syncthreads();
#pragma unroll
  for (int h = 0; h < kRows; ++h) {
    const int row = row_of(h);
    const int64_t r = (int64_t)(blockIdx.x / c.n_heads) * TILE + row;
    if (!mine[h]) continue;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      void* out = which ? rows.v : rows.k;
      const int64_t o = r * (which ? rows.ldv : rows.ldk) + head * dim;
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int d = 8 * (kLanes * i + l);
        if (d >= dim) continue;
        Piece w = raw[which][h][i];
        if (which && has[h]) {
#pragma unroll
          for (int j = 0; j < (Q4 ? 1 : (Q8 ? 2 : 4)); ++j) w[j] = values.piece(row, d)[j];
        }
        if (Q4 && has[h]) w = values4(w[0], scale4(e[which][h][i]));
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
          v[j] = Q8 ? (float)(int8_t)(w[j / 4] >> (8 * (j % 4))) * scale[which][h]
                    : __uint_as_float(j % 2 ? w[j / 2] & 0xFFFF0000u : w[j / 2] << 16);
        // past the caches, which keeps the pages in them (18829 rows, 20 heads of 64, from memory: 8-bit 30 us for 40, 4-bit 25
        // for 37, bf16 39 for 46)
        if (rows.f32) {
          typedef float Quad __attribute__((ext_vector_type(4)));
          Quad* q = reinterpret_cast<Quad*>(static_cast<float*>(out) + o + d);
          __builtin_nontemporal_store(Quad{v[0], v[1], v[2], v[3]}, q);
          __builtin_nontemporal_store(Quad{v[4], v[5], v[6], v[7]}, q + 1);
        } else {
          if (Q8) {
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = __builtin_bit_cast(uint32_t, Pair{(__bf16)v[2 * j], (__bf16)v[2 * j + 1]});
          }
          __builtin_nontemporal_store(w, reinterpret_cast<Piece*>(static_cast<uint16_t*>(out) + o + d));
        }
      }
    }
  }
}

// Tiles of 64 rows once there is one for every compute unit (24 prompts as above:
// written in 52 us, in tiles of 16 in 57), else of 16 (64 single tokens: written in
// 4.1 us, in tiles of 64 in 6.5). `launch` gets the store, the pieces of a lane and the tile's rows.
template <class Launch>
hipError_t by_kind(const KvArgs& c, const KvRowsArgs& r, Launch launch) {
  auto tile = [&](auto store, auto pieces) {
    if ((int64_t)(r.n_rows / 64) * c.n_heads >= 256) launch(store, pieces, std::integral_constant<int, 64>());
    else launch(store, pieces, std::integral_constant<int, 16>());
  };
  auto pieces = [&](auto store) {
    if (c.dim <= 64) tile(store, std::integral_constant<int, 2>());
    else if (c.dim <= 128) tile(store, std::integral_constant<int, 4>());
    else tile(store, std::integral_constant<int, 8>());
  };
  if (c.store == C4S_KV_Q8) pieces(std::integral_constant<int, C4S_KV_Q8>());
  else if (c.store == C4S_KV_Q4) pieces(std::integral_constant<int, C4S_KV_Q4>());
  else pieces(std::integral_constant<int, C4S_KV_BF16>());
  return hipGetLastError();
}

}  // namespace

hipError_t launch_kv_append(const KvArgs& c, const KvRowsArgs& r, hipStream_t s) {
  return by_kind(c, r, [&](auto store, auto pieces, auto tile) {
    constexpr int kTile = decltype(tile)::value;
    hipLaunchKernelGGL((k_kv_append<decltype(store)::value, decltype(pieces)::value, kTile>),
                       dim3((r.n_rows + kTile - 1) / kTile * c.n_heads), dim3(4 * kTile), 0, s, c, r);
  });
}

hipError_t launch_kv_read(const KvArgs& c, const KvRowsArgs& r, hipStream_t s) {
  return by_kind(c, r, [&](auto store, auto pieces, auto tile) {
    constexpr int kTile = decltype(tile)::value;
    hipLaunchKernelGGL((k_kv_read<decltype(store)::value, decltype(pieces)::value, kTile>),
                       dim3((r.n_rows + kTile - 1) / kTile * c.n_heads), dim3(4 * kTile), 0, s, c, r);
  });
}

}  // namespace c4s
