// Pages of the cache handed out, taken back and shared (include/c4s_batch.h).
//
// Handing out is one workgroup's work: sums over the sequences of the pages that
// each needs, then a walk over the words of free bits, in which every free page
// finds its number among all, and by it its sequence and table entry. Nothing
// depends on the order in which threads come, so tables are the same in every run.
// All of it is latency: a step's call is a chain of a few dependent reads.

#include <hip/hip_runtime.h>

#include <algorithm>

#include "c4s_batch.hpp"

namespace c4s {
namespace {

constexpr int kGrowThreads = 1024;

__device__ __forceinline__ int32_t count_of(const int32_t* refs, int page) {
  return __hip_atomic_load(refs + page, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// Waits until this wave's writes and atomics are done, for all that the workgroup does behind the barrier.
__device__ __forceinline__ void barrier_after_memory() {
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __builtin_amdgcn_s_waitcnt(0x0F70);   // vmcnt(0)
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __syncthreads();
}

__device__ __forceinline__ int wave_prefix(int v) {   // inclusive
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int up = __shfl_up(v, d);
    if ((int)(threadIdx.x % 64) >= d) v += up;
  }
  return v;
}

// Sums before this thread over the workgroup, and over all of it. Every thread calls it.
struct Prefix {
  int waves[2][kGrowThreads / 64];
  __device__ __forceinline__ int operator()(int v, int* total, int which) {
    const int in = wave_prefix(v), wave = threadIdx.x / 64;
    if (threadIdx.x % 64 == 63) waves[which][wave] = in;
    __syncthreads();
    int before = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < kGrowThreads / 64; ++w) {
      before += w < wave ? waves[which][w] : 0;
      sum += waves[which][w];
    }
    *total = sum;
    return before + in - v;
  }
};

__device__ __forceinline__ void drop_page(const c4s_pages& p, int page) {
  if (atomicSub(p.refs + page, 1) == 1) atomicOr(p.free_bits + page / 32, 1u << (page % 32));
}

struct GrowArgs {
  c4s_pages p;
  c4s_grow g;
  int shift;
};

__global__ __launch_bounds__(kGrowThreads) void k_pages_grow(GrowArgs f) {
  __shared__ int32_t off[kPagesSeqs + 1];   // pages asked for by the sequences before
  __shared__ int32_t last[kPagesSeqs];      // a last page that must not be written: its number; -1: none
  __shared__ Prefix prefix;
  __shared__ int any_shared;
  const c4s_pages& p = f.p;
  const c4s_grow& g = f.g;
  const int tid = threadIdx.x, n = p.n_seqs, shift = f.shift, ps = 1 << shift;
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
  };
  load_bits(4 * tid);

  auto pages_of = [&](int64_t tokens) { return (int)min((tokens + ps - 1) >> shift, (int64_t)p.max_pages); };
  auto news_of = [&](int b) { return g.n_new ? max(g.n_new[b], 0) : 1; };
  auto len_of = [&](int b) { return max(p.lens[b], 0); };

  if (g.copies) {
    if (tid == 0) any_shared = 0;
    __syncthreads();
    for (int b = tid; b < n; b += kGrowThreads) {
      const int len = len_of(b), at = len >> shift;
      int page = -1;
      if ((len & (ps - 1)) && at < p.max_pages && news_of(b) > 0) {
        page = p.block_table[b * p.table_ld + at];
        if (page < 0 || page >= p.n_pages || count_of(p.refs, page) < 2) page = -1;
      }
      last[b] = page;
      if (page >= 0) any_shared = 1;
      reinterpret_cast<int2*>(g.copies)[b] = make_int2(-1, -1);
    }
    __syncthreads();
    if (any_shared) {
      // Every sharer gives up its hold; a page that none is left of stays with the last of them, whose
      // number (+ 1) is the largest that the count is raised to.
      for (int b = tid; b < n; b += kGrowThreads)
        if (last[b] >= 0) atomicSub(p.refs + last[b], 1);
      barrier_after_memory();
      for (int b = tid; b < n; b += kGrowThreads) {   // kept by others: 0 .. - 1 is no page and stays so
        const int page = last[b];
        if (page >= 0 && count_of(p.refs, page) != 0) last[b] = page | 1 << 30;
      }
      barrier_after_memory();
      for (int b = tid; b < n; b += kGrowThreads)
        if (last[b] >= 0 && !(last[b] >> 30)) atomicMax(p.refs + last[b], b + 1);
      barrier_after_memory();
      for (int b = tid; b < n; b += kGrowThreads)
        if (last[b] >= 0 && !(last[b] >> 30) && count_of(p.refs, last[b]) == b + 1) last[b] = -2 - last[b];
      barrier_after_memory();
      for (int b = tid; b < n; b += kGrowThreads) {
        if (last[b] < -1) {
          __hip_atomic_store(p.refs - 2 - last[b], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          last[b] = -1;
        } else if (last[b] >= 0) {
          last[b] &= (1 << 30) - 1;
        }
      }
    }
  } else {
    for (int b = tid; b < n; b += kGrowThreads) last[b] = -1;
  }

  int64_t rows = 0;   // of the sequences before these
  int asked = 0;
  int lost = 0;       // pages behind the table's end
  for (int b0 = 0; b0 < n; b0 += kGrowThreads) {
    const int b = b0 + tid;
    int need = 0, fresh = 0;
    int64_t len = 0;
    if (b < n) {
      len = len_of(b);
      fresh = news_of(b);
      const int64_t whole = (len + fresh + ps - 1) >> shift;
      need = pages_of(len + fresh) - pages_of(len) + (last[b] >= 0);
      lost += (int)(whole - ((len + ps - 1) >> shift) - (pages_of(len + fresh) - pages_of(len)));
    }
    int sum;
    const int before = prefix(need, &sum, 0);
    if (b < n) off[b] = asked + before;
    asked += sum;
    if (g.rows_off) {
      int fresh_sum;
      const int fresh_before = prefix(fresh, &fresh_sum, 1);
      if (b < n) g.rows_off[b] = (int32_t)(rows + fresh_before);
      rows += fresh_sum;
    }
    __syncthreads();
  }
  if (tid == 0) {
    off[n] = asked;
    if (g.rows_off) g.rows_off[n] = (int32_t)rows;
  }
  __syncthreads();

  // Table entry number `rank` of those asked for.
  auto give = [&](int rank, int page) {
    int lo = 0, hi = n;   // the last sequence that begins at or before it (those that ask for none begin with the next)
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (off[mid] <= rank) lo = mid;
      else hi = mid;
    }
    const int own = last[lo] >= 0, nth = rank - off[lo], len = len_of(lo);
    const int at = own && nth == 0 ? len >> shift : pages_of(len) + nth - own;
    p.block_table[lo * p.table_ld + at] = page;
    if (own && nth == 0 && page >= 0) reinterpret_cast<int2*>(g.copies)[lo] = make_int2(last[lo], page);
  };
  int found = 0;
  for (int w0 = 0; w0 < words && found < asked; w0 += 4 * kGrowThreads) {
    const int word = w0 + 4 * tid;
    if (w0) load_bits(word);
    uint32_t v[4] = {bits.x, bits.y, bits.z, bits.w};
    int sum;
    int rank = found + prefix(__popc(v[0]) + __popc(v[1]) + __popc(v[2]) + __popc(v[3]), &sum, w0 / (4 * kGrowThreads) & 1);
    found += sum;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t left = v[i];
      while (left && rank < asked) {
        const int page = 32 * (word + i) + __ffs(left) - 1;
        left &= left - 1;
        if (page >= p.n_pages) break;
        p.refs[page] = 1;
        give(rank++, page);
      }
      if (left != v[i]) p.free_bits[word + i] = left;
    }
  }
  for (int rank = found + tid; rank < asked; rank += kGrowThreads) give(rank, -1);
  if (p.missing) {
    if (lost) atomicAdd(p.missing, lost);
    if (tid == 0 && asked > found) atomicAdd(p.missing, asked - found);
  }
  barrier_after_memory();   // every table entry is written, every length read
  for (int b = tid; b < n; b += kGrowThreads) {
    const int len = len_of(b), fresh = news_of(b);
    p.lens[b] = (int32_t)min((int64_t)len + fresh, (int64_t)INT32_MAX);
    if (!g.n_new && b < g.n_rows) {   // row b: the sequence's one new token
      if (g.row_pos) g.row_pos[b] = len;
      if (g.row_slot) {
        const int at = len >> shift, page = at < p.max_pages ? p.block_table[b * p.table_ld + at] : -1;
        g.row_slot[b] = page < 0 || page >= p.n_pages ? -1 : (page << shift) + (len & (ps - 1));
      }
    }
  }
}

// Rows of several new tokens a sequence: positions and slots.
__global__ __launch_bounds__(256) void k_row_maps(GrowArgs f) {
  const c4s_pages& p = f.p;
  const c4s_grow& g = f.g;
  const int r = blockIdx.x * 256 + threadIdx.x;
  if (r >= g.n_rows || r >= g.rows_off[p.n_seqs]) return;
  int lo = 0, hi = p.n_seqs;
  while (hi - lo > 1) {
    const int step = (hi - lo + 7) / 8;
    int behind = 0;
#pragma unroll
    for (int j = 1; j < 8; ++j) behind += (lo + j * step < hi) & (g.rows_off[min(lo + j * step, hi - 1)] <= r);
    lo += behind * step;
    hi = min(lo + step, hi);
  }
  const int pos = p.lens[lo] - (g.rows_off[lo + 1] - r), at = pos >> f.shift;
  if (g.row_pos) g.row_pos[r] = pos;
  if (!g.row_slot) return;
  const int page = at < p.max_pages ? p.block_table[lo * p.table_ld + at] : -1;
  g.row_slot[r] = page < 0 || page >= p.n_pages ? -1 : (page << f.shift) + (pos & ((1 << f.shift) - 1));
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
  const char* tensor[4];   // keys, values and their scales; bytes of a page of each, all multiples of 16
  uint32_t units[4];       // of 16 bytes
  const int32_t* copies;
  int n_pages;
};

// A workgroup copies a part of a pair's 16-byte units, four of a thread's in flight.
__global__ __launch_bounds__(256) void k_kv_copy(CopyArgs f) {
  const int2 pair = reinterpret_cast<const int2*>(f.copies)[blockIdx.y];
  if (pair.x < 0 || pair.x >= f.n_pages || pair.y < 0 || pair.y >= f.n_pages || pair.x == pair.y) return;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const uint32_t n = f.units[t];
    const uint4* from = reinterpret_cast<const uint4*>(f.tensor[t]) + (uint64_t)pair.x * n;
    uint4* to = reinterpret_cast<uint4*>(const_cast<char*>(f.tensor[t])) + (uint64_t)pair.y * n;
    const uint32_t step = 256 * gridDim.x;
    for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < n; i += 4 * step) {
      uint4 v[4];
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j)
        if (i + j * step < n) v[j] = from[i + j * step];
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j)
        if (i + j * step < n) to[i + j * step] = v[j];
    }
  }
}

int shift_of(int page_size) {
  int s = 0;
  while ((1 << s) < page_size) ++s;
  return s;
}

}  // namespace

hipError_t launch_pages_grow(const c4s_pages& p, const c4s_grow& g, hipStream_t s) {
  const GrowArgs f{p, g, shift_of(p.page_size)};
  hipLaunchKernelGGL(k_pages_grow, dim3(1), dim3(kGrowThreads), 0, s, f);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || !g.n_new || g.n_rows == 0 || (!g.row_pos && !g.row_slot)) return e;
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
  const CopyArgs f{{static_cast<const char*>(c.k), static_cast<const char*>(c.v), reinterpret_cast<const char*>(c.k_scale),
                    reinterpret_cast<const char*>(c.v_scale)}, {a, a, b, b}, copies, c.n_pages};
  // a part is 1024 units of the keys, up to as many parts as a grid has room for
  hipLaunchKernelGGL(k_kv_copy, dim3(std::min<uint32_t>((a + 1023) / 1024, 4096), n), dim3(256), 0, s, f);
  return hipGetLastError();
}

}  // namespace c4s
