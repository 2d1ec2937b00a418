// mbarriers and asynchronous copies for the kernels of the paged 8-bit cache.
// Every wait is bounded: one that runs out sets the block's stop word and the
// status word, and the kernel ends.
#pragma once

#include "kv8.cuh"

namespace kv8 {

constexpr unsigned long long WAIT_NS = EMMY_KV8_WAIT_NS;

__device__ __forceinline__ uint32_t smem_addr(const void *p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void bar_init(uint64_t *b, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(b)), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t *b) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(b)) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t b, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(b), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ unsigned long long now_ns() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
// Waits with a whole warp, which stays converged, for the phase of parity
// `parity`; false when the kernel gives up, after `limit` ns.
__device__ __forceinline__ bool warp_wait(uint64_t *b, uint32_t parity, volatile unsigned *stop,
                                          unsigned *status, unsigned long long limit) {
  const uint32_t at = smem_addr(b);
  if (__all_sync(0xffffffffu, bar_try(at, parity))) return true;
  const unsigned long long t0 = now_ns();
  for (;;) {
    if (__all_sync(0xffffffffu, bar_try(at, parity))) return true;
    bool over = *stop != 0;
    if (now_ns() - t0 > limit) {
      *stop = 1;
      report(status, STATUS_WAIT);
      over = true;
    }
    if (__any_sync(0xffffffffu, over)) return false;
  }
}
// Every lane's earlier work is done: one arrival for the warp.
__device__ __forceinline__ void warp_arrive(uint64_t *b) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) bar_arrive(b);
}
__device__ __forceinline__ uint32_t elected() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r;
}

// All threads of the cluster: what each wrote before is visible after.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// The same place of this block's shared memory in block `rank` of the cluster.
__device__ __forceinline__ uint32_t peer_addr(const void *mine, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr(mine)), "r"(rank));
  return r;
}
__device__ __forceinline__ float peer_load(uint32_t at) {
  float x;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(at) : "memory");
  return x;
}
__device__ __forceinline__ float4 peer_load4(uint32_t at) {
  float4 x;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w)
               : "r"(at)
               : "memory");
  return x;
}

// A ring of n slots: slot and phase of step after step.
struct Ring {
  int slot = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next(int n) {
    if (++slot == n) slot = 0, phase ^= 1;
  }
};

}  // namespace kv8
