// Pages of the cache handed out, taken back and shared (include/c4s_batch.h).
//
// Handing out is one workgroup's work: sums over the sequences of the pages that
// each needs, then a walk over the words of free bits, in which every free page
// finds its number among all. The pages pass through LDS in that order, so that
// all threads share in handing them out. (1000 sequences' 17000 pages take 25 us, the
// 150 of 256 beams, all from a few words, 9.6; with each thread handing out what its
// words hold 71 and 52.)
// Who shares a last page with whom is found in a hash table in LDS. Nothing depends on
// the order in which threads come, so tables are the same in every run.
// A step's call is a chain of a few dependent reads (64 sequences: 8.5 us, 2.7 of them
// the launch; a trim 3.6, a fork of 64 groups of 4 5.4). With thousands of pages, too, its waves
// wait for half of the time: VALU 57 % busy, LDS 23 %.

#include <hip/hip_runtime.h>

#include <algorithm>

#include "c4s_batch.hpp"

namespace c4s {
namespace {

constexpr int kGrowThreads = 1024;

__device__ __forceinline__ int wave_prefix(int v) {   // inclusive
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int up = __shfl_up(v, d);
    if ((int)(threadIdx.x % 64) >= d) v += up;
  }
  return v;
}

// Sums before this thread over the workgroup, and over all of it, of two numbers. Every thread calls it, and
// between two calls with one `which` there is a barrier.
struct Prefix {
  int2 waves[2][kGrowThreads / 64];
  __device__ __forceinline__ int2 operator()(int2 v, int2* total, int which) {
    const int2 in = make_int2(wave_prefix(v.x), wave_prefix(v.y));
    const int wave = threadIdx.x / 64;
    if (threadIdx.x % 64 == 63) waves[which][wave] = in;
    __syncthreads();
    int2 before = make_int2(0, 0), sum = before;
#pragma unroll
    for (int w = 0; w < kGrowThreads / 64; ++w) {
      const int2 o = waves[which][w];
      before.x += w < wave ? o.x : 0;
      before.y += w < wave ? o.y : 0;
      sum.x += o.x;
      sum.y += o.y;
    }
    *total = sum;
    return make_int2(before.x + in.x - v.x, before.y + in.y - v.y);
  }
};

__device__ __forceinline__ void drop_page(const c4s_pages& p, int page) {
  if (atomicSub(p.refs + page, 1) == 1) atomicOr(p.free_bits + page / 32, 1u << (page % 32));
}

struct GrowArgs {
  c4s_pages p;
  c4s_grow g;
  int shift;
  bool maps;   // the new rows' maps are the one workgroup's work too
};

// Position and slot of row r, the sequences' first rows at off.
__device__ __forceinline__ void map_row(const GrowArgs& f, const int32_t* off, int r) {
  const c4s_pages& p = f.p;
  int lo = 0, hi = p.n_seqs;
  while (hi - lo > 1) {   // eight parts a step
    const int step = (hi - lo + 7) / 8;
    int behind = 0;
#pragma unroll
    for (int j = 1; j < 8; ++j) behind += (lo + j * step < hi) & (off[min(lo + j * step, hi - 1)] <= r);
    lo += behind * step;
    hi = min(lo + step, hi);
  }
  const int pos = p.lens[lo] - (off[lo + 1] - r), at = pos >> f.shift;
  if (f.g.row_pos) f.g.row_pos[r] = pos;
  if (!f.g.row_slot) return;
  const int page = pos >= 0 && at < p.max_pages ? p.block_table[lo * p.table_ld + at] : -1;
  f.g.row_slot[r] = page < 0 || page >= p.n_pages ? -1 : (page << f.shift) + (pos & ((1 << f.shift) - 1));
}

constexpr int kHash = 2 * kPagesSeqs;   // places of the table of shared pages
constexpr int kBatch = 16384;           // pages in LDS at a time
// Rows whose maps that workgroup writes; more have a kernel of their own. 64 sequences, new tokens each, with a trim,
// us: 16 11.3 (own kernel 12.2), 32 12.9 (13.4), 64 16.7 (14.9), 256 32 (18.6).
constexpr int kMapRows = 2048;

__global__ __launch_bounds__(kGrowThreads) void k_pages_grow(GrowArgs f) {
  __shared__ union {
    struct {
      int32_t page[kHash], users[kHash], last[kHash];   // a shared page (-1: none), how many go on, the last of them
    } hash;
    struct {
      int32_t off[kPagesSeqs + 1];   // pages asked for by the sequences before
      int32_t page[kBatch];          // free pages in order
      uint4 words[kGrowThreads];     // the free bits that are looked at,
      int32_t before[kGrowThreads];  // and how many free pages lie before each four words
    } give;
  } lds;
  __shared__ int32_t lens[kPagesSeqs];
  __shared__ int32_t here[kPagesSeqs];    // the page of a sequence's first new token, where there is one
  __shared__ int32_t old[kPagesSeqs];     // a last page that must not be written; -1: none
  __shared__ Prefix prefix;
  const c4s_pages& p = f.p;
  const c4s_grow& g = f.g;
  const int tid = threadIdx.x, lane = tid % 64, n = p.n_seqs, shift = f.shift, ps = 1 << shift;
  const int words = (p.n_pages + 31) / 32;
  // the free bits' first words are underway while the sequences are looked at
  uint4 bits = make_uint4(0, 0, 0, 0);
  auto load_bits = [&](int word) {
    bits = make_uint4(0, 0, 0, 0);
    if (word + 4 <= words) bits = *reinterpret_cast<const uint4*>(p.free_bits + word);
    else {
      if (word < words) bits.x = p.free_bits[word];
      if (word + 1 < words) bits.y = p.free_bits[word + 1];
      if (word + 2 < words) bits.z = p.free_bits[word + 2];
    }
    const int last = words - 1 - word;   // bits behind the last page count for nothing
    if (last >= 0 && last < 4 && p.n_pages % 32) (last == 0 ? bits.x : last == 1 ? bits.y : last == 2 ? bits.z : bits.w) &= (1u << p.n_pages % 32) - 1;
  };
  load_bits(4 * tid);

  auto pages_of = [&](int64_t tokens) { return (int)min((tokens + ps - 1) >> shift, (int64_t)p.max_pages); };
  auto news_of = [&](int b) { return g.n_new ? max(g.n_new[b], 0) : 1; };
  auto is_page = [&](int page) { return page >= 0 && page < p.n_pages; };

  if (g.copies)
    for (int i = tid; i < kHash; i += kGrowThreads) lds.hash.page[i] = -1, lds.hash.users[i] = 0, lds.hash.last[i] = -1;
  for (int b = tid; b < n; b += kGrowThreads) {
    const int len = max(p.lens[b], 0), at = len >> shift;
    lens[b] = len;
    here[b] = (len & (ps - 1)) && at < p.max_pages ? p.block_table[b * p.table_ld + at] : -1;
    old[b] = -1;
  }
  if (g.copies) {
    // Pages of several holders that are about to be written: who has them, and of those who go on the last. If they
    // are all the holders, the last keeps the page; the others give up their hold on it.
    __syncthreads();
    constexpr int kMine = kPagesSeqs / kGrowThreads;
    int place[kMine], holders[kMine];
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int b = tid + i * kGrowThreads;
      place[i] = -1;
      holders[i] = 0;
      if (b < n && is_page(here[b]) && news_of(b) > 0) holders[i] = p.refs[here[b]];
    }
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      if (holders[i] < 2) continue;
      const int b = tid + i * kGrowThreads, page = here[b];
      int at = (int)((uint32_t)page * 2654435761u >> 19);   // 13 bits
      static_assert(kHash == 1 << 13, "the hash's bits");
      for (;;) {   // there are more places than sequences
        const int was = atomicCAS(&lds.hash.page[at], -1, page);
        if (was == -1 || was == page) break;
        at = (at + 1) % kHash;
      }
      place[i] = at;
      atomicAdd(&lds.hash.users[at], 1);
      atomicMax(&lds.hash.last[at], b);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int b = tid + i * kGrowThreads;
      if (b >= n) break;
      reinterpret_cast<int2*>(g.copies)[b] = make_int2(-1, -1);
      if (place[i] < 0 || (lds.hash.users[place[i]] == holders[i] && lds.hash.last[place[i]] == b)) continue;
      old[b] = here[b];
      here[b] = -1;
      atomicSub(p.refs + old[b], 1);
    }
  }
  __syncthreads();

  int64_t rows = 0;   // of the sequences before these
  int asked = 0;
  int lost = 0;       // pages behind the table's end
  for (int b0 = 0; b0 < n; b0 += kGrowThreads) {
    const int b = b0 + tid;
    int need = 0, fresh = 0;
    if (b < n) {
      const int64_t len = lens[b];
      fresh = news_of(b);
      const int more = pages_of(len + fresh) - pages_of(len);
      need = more + (old[b] >= 0);
      lost += (int)(((len + fresh + ps - 1) >> shift) - ((len + ps - 1) >> shift)) - more;
    }
    int2 sum;
    const int2 before = prefix(make_int2(need, fresh), &sum, 0);
    if (b < n) {
      lds.give.off[b] = asked + before.x;
      if (g.rows_off) g.rows_off[b] = (int32_t)(rows + before.y);
    }
    asked += sum.x;
    rows += sum.y;
    __syncthreads();
  }
  if (tid == 0) {
    lds.give.off[n] = asked;
    if (g.rows_off) g.rows_off[n] = (int32_t)rows;
  }
  __syncthreads();

  // The pages asked for from number `first` on, `count` of them, -1 where there are none, into sequence b's entries:
  // those with numbers begin .. end - 1 and every step-th.
  auto put = [&](int b, int begin, int end, int step, int first, bool there) {
    const int off = lds.give.off[b], own = old[b] >= 0, len = lens[b];
    int32_t* row = p.block_table + b * p.table_ld;
    if (begin >= end) return;
    if (begin == off) {
      const int page = there ? lds.give.page[begin - first] : -1;
      here[b] = page;
      if (own) {
        row[len >> shift] = page;
        if (page >= 0) reinterpret_cast<int2*>(g.copies)[b] = make_int2(old[b], page);
        begin += step;
      }
    }
    row += pages_of(len) - own - off;
    for (int rank = begin; rank < end; rank += step) row[rank] = there ? lds.give.page[rank - first] : -1;
  };
  // Few: a page a thread, which searches its sequence; many: sixteen threads a sequence, which write its entries next to
  // each other. (4000 sequences, one page each, with a trim: 35 us, by sixteen 51; 1000 of three 27 and 29, of 13 39 and 31.)
  auto give = [&](int first, int count, bool there) {
    if (count <= 2 * kGrowThreads || count <= 4 * n) {
      for (int i = tid; i < count; i += kGrowThreads) {
        int lo = 0, hi = n;   // the last sequence that begins at or before it (those that ask for none begin with the next)
        while (hi - lo > 1) {
          const int mid = (lo + hi) / 2;
          if (lds.give.off[mid] <= first + i) lo = mid;
          else hi = mid;
        }
        put(lo, first + i, first + i + 1, 1, first, there);
      }
    } else {
      for (int b = tid / 16; b < n; b += kGrowThreads / 16)
        put(b, max(lds.give.off[b], first) + tid % 16, min(lds.give.off[b + 1], first + count), 16, first, there);
    }
  };
  int found = 0;
  for (int w0 = 0, turn = 0; w0 < words && found < asked; w0 += 4 * kGrowThreads, ++turn) {
    const int word = w0 + 4 * tid;
    uint32_t v[4] = {bits.x, bits.y, bits.z, bits.w};
    if (w0 + 4 * kGrowThreads < words) load_bits(word + 4 * kGrowThreads);
    int2 sum;
    const int mine = found + prefix(make_int2(__popc(v[0]) + __popc(v[1]) + __popc(v[2]) + __popc(v[3]), 0), &sum, turn & 1).x;
    const int upto = min(found + sum.x, asked);
    lds.give.words[tid] = make_uint4(v[0], v[1], v[2], v[3]);
    lds.give.before[tid] = mine;
    __syncthreads();
    for (int first = found; first < upto; first += kBatch) {
      const int count = min(upto - first, kBatch);
      // a wave takes every sixteenth four words, two at a time, a lane a bit (a thread on its own words' bits would write
      // as many places apart: all lanes in one bank)
      constexpr int kWaves = kGrowThreads / 64;
      const int q = lane * kWaves + tid / 64, q_before = lds.give.before[q], q_next = q + 1 < kGrowThreads ? lds.give.before[q + 1] : found + sum.x;
      uint64_t lanes = __ballot(q_before < first + count && q_next > first);
      while (lanes) {
        const int l = __ffsll((unsigned long long)lanes) - 1, at4 = l * kWaves + tid / 64;
        lanes &= lanes - 1;
        const uint4 w = lds.give.words[at4];
        int rank = lds.give.before[at4] - first;
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          const uint64_t pair = i ? (uint64_t)w.w << 32 | w.z : (uint64_t)w.y << 32 | w.x;
          const int at = rank + __popcll(pair & ((1ull << lane) - 1));
          if ((pair >> lane & 1) && at >= 0 && at < count) lds.give.page[at] = 32 * (w0 + 4 * at4 + i) + lane;
          rank += __popcll(pair);
        }
      }
      __syncthreads();
      for (int i = tid; i < count; i += kGrowThreads) p.refs[lds.give.page[i]] = 1;
      give(first, count, true);
      __syncthreads();
    }
    int rank = mine;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int have = __popc(v[i]), taken = min(max(upto - rank, 0), have);
      rank += have;
      if (!taken) continue;
      uint32_t left = taken == have ? 0 : v[i];
      for (int t = 0; left && t < taken; ++t) left &= left - 1;
      p.free_bits[word + i] = left;
    }
    found += sum.x;
  }
  if (found < asked) give(found, asked - found, false);
  if (p.missing) {
    if (lost) atomicAdd(p.missing, lost);
    if (tid == 0 && asked > found) atomicAdd(p.missing, asked - found);
  }
  __syncthreads();
  for (int b = tid; b < n; b += kGrowThreads) {
    const int len = lens[b];
    p.lens[b] = (int32_t)min((int64_t)len + news_of(b), (int64_t)INT32_MAX);
    if (!g.n_new && b < g.n_rows) {   // row b: the sequence's one new token
      if (g.row_pos) g.row_pos[b] = len;
      if (g.row_slot) g.row_slot[b] = is_page(here[b]) ? (here[b] << shift) + (len & (ps - 1)) : -1;
    }
  }
  if (!f.maps) return;
  int32_t* off = lds.give.page;   // (no page is handed out any more)
  static_assert(kPagesSeqs < kBatch, "the rows' offsets in LDS");
  for (int b = tid; b <= n; b += kGrowThreads) off[b] = g.rows_off[b];
  __syncthreads();
  for (int row = tid; row < min(g.n_rows, off[n]); row += kGrowThreads) map_row(f, off, row);
}

// Rows of several new tokens a sequence: positions and slots.
__global__ __launch_bounds__(256) void k_row_maps(GrowArgs f) {
  const int r = blockIdx.x * 256 + threadIdx.x;
  if (r < f.g.n_rows && r < f.g.rows_off[f.p.n_seqs]) map_row(f, f.g.rows_off, r);
}

// A wave a sequence.
__global__ __launch_bounds__(256) void k_pages_trim(c4s_pages p, const int32_t* n_drop, int shift) {
  const int b = blockIdx.x * 4 + threadIdx.x / 64, lane = threadIdx.x % 64, ps = 1 << shift;
  if (b >= p.n_seqs) return;
  const int len = max(p.lens[b], 0), drop = min(max(n_drop[b], 0), len);
  if (drop == 0) return;
  const int from = (int)(((int64_t)(len - drop) + ps - 1) >> shift), to = (int)min(((int64_t)len + ps - 1) >> shift, (int64_t)p.max_pages);
  for (int i = from + lane; i < to; i += 64) {
    int32_t* entry = p.block_table + b * p.table_ld + i;
    const int page = *entry;
    *entry = -1;
    if (page >= 0 && page < p.n_pages) drop_page(p, page);
  }
  if (lane == 0) p.lens[b] = len - drop;
}

constexpr int kForkThreads = 256;

// A workgroup has a group's rows over 256 entries; a thread reads one entry of every row before it writes any.
// Of a row with c children a page's count changes by c - 1, in one addition: a count that passes 0 on its way
// has lost every holder, so it stays there, and the one addition that reached it frees the page.
__global__ __launch_bounds__(kForkThreads) void k_pages_fork(c4s_pages p, const int32_t* parent, int width) {
  __shared__ int32_t mine[kBeamWidth][kForkThreads];
  __shared__ int from[kBeamWidth], children[kBeamWidth];
  const int tid = threadIdx.x, base = blockIdx.y * width, at = blockIdx.x * kForkThreads + tid;
  if (tid < width) children[tid] = 0;
  __syncthreads();
  if (tid < width) {
    const int j = parent[base + tid];
    from[tid] = j >= 0 && j < width ? j : -1;
    if (from[tid] >= 0) atomicAdd(&children[from[tid]], 1);
  }
  int len = 0;
  __syncthreads();
  if (blockIdx.x == 0 && tid < width && from[tid] >= 0) len = p.lens[base + from[tid]];
  __syncthreads();
  if (blockIdx.x == 0 && tid < width) p.lens[base + tid] = len;
  if (at >= p.max_pages) return;
  for (int j = 0; j < width; ++j) mine[j][tid] = p.block_table[(base + j) * p.table_ld + at];
  for (int j = 0; j < width; ++j) {
    const int page = mine[j][tid], more = children[j] - 1;
    if (page >= 0 && page < p.n_pages && more) {
      if (atomicAdd(p.refs + page, more) + more == 0) atomicOr(p.free_bits + page / 32, 1u << (page % 32));
    }
    p.block_table[(base + j) * p.table_ld + at] = from[j] < 0 ? -1 : mine[from[j]][tid];
  }
}

// ---- pages copied ---------------------------------------------------------------------

struct CopyArgs {
  char* tensor[4];         // keys, values and their scales
  uint32_t begin[5];       // their units of 16 bytes in a page, one behind the other
  const int32_t* copies;
  int n_pages;
};

typedef uint32_t Unit __attribute__((ext_vector_type(4)));

// A workgroup copies 1024 of a pair's units, a thread's four together on their way (96 pages of 21 KB: 3.7 us; a unit of a
// thread at a time 12).
__global__ __launch_bounds__(256) void k_kv_copy(CopyArgs f) {
  const int2 pair = reinterpret_cast<const int2*>(f.copies)[blockIdx.y];
  if (pair.x < 0 || pair.x >= f.n_pages || pair.y < 0 || pair.y >= f.n_pages || pair.x == pair.y) return;
  for (uint32_t first = blockIdx.x * 1024; first < f.begin[4]; first += 1024 * gridDim.x) {
    Unit v[4];
    char* to[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t i = first + 256 * j + threadIdx.x;
      const bool there = i < f.begin[4];   // (else the first unit, which is not written)
      const int t = there ? (i >= f.begin[1]) + (i >= f.begin[2]) + (i >= f.begin[3]) : 0;
      const uint32_t begin = t == 0 ? 0 : (t == 1 ? f.begin[1] : (t == 2 ? f.begin[2] : f.begin[3]));
      const uint32_t end = t == 0 ? f.begin[1] : (t == 1 ? f.begin[2] : (t == 2 ? f.begin[3] : f.begin[4]));
      char* tensor = t == 0 ? f.tensor[0] : (t == 1 ? f.tensor[1] : (t == 2 ? f.tensor[2] : f.tensor[3]));
      const uint64_t bytes = 16ull * (end - begin), at = there ? 16ull * (i - begin) : 0;
      v[j] = *reinterpret_cast<const Unit*>(tensor + pair.x * bytes + at);
      to[j] = there ? tensor + pair.y * bytes + at : nullptr;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (to[j]) *reinterpret_cast<Unit*>(to[j]) = v[j];
  }
}

int shift_of(int page_size) {
  int s = 0;
  while ((1 << s) < page_size) ++s;
  return s;
}

}  // namespace

hipError_t launch_pages_grow(const c4s_pages& p, const c4s_grow& g, hipStream_t s) {
  const bool maps = g.n_new && g.n_rows && (g.row_pos || g.row_slot);
  const GrowArgs f{p, g, shift_of(p.page_size), maps && g.n_rows <= kMapRows};
  hipLaunchKernelGGL(k_pages_grow, dim3(1), dim3(kGrowThreads), 0, s, f);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || !maps || f.maps) return e;
  hipLaunchKernelGGL(k_row_maps, dim3((g.n_rows + 255) / 256), dim3(256), 0, s, f);
  return hipGetLastError();
}

hipError_t launch_pages_trim(const c4s_pages& p, const int32_t* n_drop, hipStream_t s) {
  hipLaunchKernelGGL(k_pages_trim, dim3((p.n_seqs + 3) / 4), dim3(256), 0, s, p, n_drop, shift_of(p.page_size));
  return hipGetLastError();
}

hipError_t launch_pages_fork(const c4s_pages& p, const int32_t* parent, int width, hipStream_t s) {
  hipLaunchKernelGGL(k_pages_fork, dim3(std::max((p.max_pages + kForkThreads - 1) / kForkThreads, 1), p.n_seqs / width),
                     dim3(kForkThreads), 0, s, p, parent, width);
  return hipGetLastError();
}

hipError_t launch_kv_copy(const KvArgs& c, const int32_t* copies, int n, hipStream_t s) {
  const uint64_t values = (uint64_t)c.n_heads * c.dim << c.page_shift, rows = (uint64_t)c.n_heads << c.page_shift;
  const uint64_t page = c.store == C4S_KV_BF16 ? 2 * values : (c.store == C4S_KV_Q8 ? values : values / 2);
  const uint64_t scales = c.store == C4S_KV_BF16 ? 0 : (c.store == C4S_KV_Q8 ? 4 * rows : rows * (c.dim / 32));
  const uint32_t a = (uint32_t)(page / 16), b = (uint32_t)(scales / 16);
  const CopyArgs f{{static_cast<char*>(c.k), static_cast<char*>(c.v), reinterpret_cast<char*>(c.k_scale), reinterpret_cast<char*>(c.v_scale)},
                   {0, a, 2 * a, 2 * a + b, 2 * a + 2 * b}, copies, c.n_pages};
  hipLaunchKernelGGL(k_kv_copy, dim3(std::min<uint32_t>((2 * a + 2 * b + 1023) / 1024, 4096), n), dim3(256), 0, s, f);
  return hipGetLastError();
}

}  // namespace c4s
