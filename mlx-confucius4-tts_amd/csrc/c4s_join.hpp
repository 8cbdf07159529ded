// Parts of one result from several workgroups, joined by the last of them to
// arrive (device side).
//
// The workgroups may sit on different XCDs, whose L2s do not see each other's
// lines. The usual way, an agent-scope release fence, writes back everything
// the XCD's L2 holds: with 240 workgroups it took 25 us. The parts are instead written and
// read past the L2s, as relaxed agent-scope atomics of 8 bytes, and a store
// counts as done (vmcnt) once it is where every XCD sees it: each wave waits
// for its own, the barrier collects the waves, and only then does one thread
// count the workgroup in.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace c4s {

typedef float f32x4 __attribute__((ext_vector_type(4)));

// A part is n quads of floats, thread by thread: quad q's first half is 8-byte
// word q and its second word n + q, so that a wave's stores are contiguous.
__device__ __forceinline__ void put_quad(float* part, int n, int q, f32x4 v) {
  const uint4 w = __builtin_bit_cast(uint4, v);
  uint64_t* p = reinterpret_cast<uint64_t*>(part) + q;
  __hip_atomic_store(p, (uint64_t)w.y << 32 | w.x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __hip_atomic_store(p + n, (uint64_t)w.w << 32 | w.z, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ f32x4 get_quad(const float* part, int n, int q) {
  const uint64_t* p = reinterpret_cast<const uint64_t*>(part) + q;
  const uint64_t a = __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  const uint64_t b = __hip_atomic_load(p + n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return __builtin_bit_cast(f32x4, make_uint4((uint32_t)a, (uint32_t)(a >> 32), (uint32_t)b, (uint32_t)(b >> 32)));
}

// Whether this workgroup is the last of `n` to arrive; the same for all its
// threads, which have all put their parts. The last leaves the counter zero.
__device__ __forceinline__ bool last_to_arrive(uint32_t* counter, int n) {
  __shared__ bool last;
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __builtin_amdgcn_s_waitcnt(0x0F70);   // vmcnt(0): this wave's parts are out
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __syncthreads();
  if (threadIdx.x == 0) {
    last = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)n - 1;
    if (last) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  return last;
}

}  // namespace c4s
