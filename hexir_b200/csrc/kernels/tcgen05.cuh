// tcgen05.cuh -- the fifth-generation tensor core instructions the 16-bit
// products use (linear_16.cu): TMEM allocation, shared-memory and
// instruction descriptors, the MMA, its commit, and TMEM loads.  CG is the
// CTA group: 1, or 2 for a pair of CTAs that compute one tile.
#pragma once

#include "common.cuh"

namespace hexir {

// mbar_wait_bounded for the main loops: `tried` says that the phase was seen
// complete already (a try issued earlier, whose answer took its ~100 cycles
// under other work).  The timer is read only after 64 tries.
__device__ __forceinline__ bool mbar_wait_pipeline(uint64_t *bar, uint32_t parity,
                                                   uint64_t timeout_ns,
                                                   bool tried = false) {
  if (tried)
    return true;
  uint64_t start = 0;
  for (uint32_t spin = 1;; ++spin) {
    if (mbar_try_wait(bar, parity))
      return true;
    if ((spin & 63u) == 0u) {
      const uint64_t now = global_timer_ns();
      if (start == 0) {
        start = now;
      } else if (now - start > timeout_ns) {
        atomicOr(&hexir_device_error_word, HEXIR_KERR_WAIT_TIMEOUT);
        return false;
      }
    }
  }
}

// Whether the phase with the given parity has completed, without waiting (a
// try_wait may hold the thread for a while).
__device__ __forceinline__ bool mbar_test(uint64_t *bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(smem_addr(bar)), "r"(parity)
      : "memory");
  return done != 0;
}

// One lane of a converged warp, the same at every call.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xFFFFFFFF;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(p));
  return p != 0;
}

// A place in a ring of stages: the stage, and the parity of its use.
struct RingPlace {
  uint32_t stage = 0, parity = 0;
  __device__ __forceinline__ void next(uint32_t stages) {
    if (++stage == stages) {
      stage = 0;
      parity ^= 1u;
    }
  }
};

template <int CG>
__device__ __forceinline__ void tmem_alloc(uint32_t *slot, uint32_t cols) {
  if (CG == 1) {
    asm volatile(
        "tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
            smem_addr(slot)),
        "r"(cols)
        : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  } else {
    asm volatile(
        "tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
            smem_addr(slot)),
        "r"(cols)
        : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
}

template <int CG>
__device__ __forceinline__ void tmem_free(uint32_t tmem, uint32_t cols) {
  if (CG == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(
                     tmem),
                 "r"(cols));
  else
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(
                     tmem),
                 "r"(cols));
}

__device__ __forceinline__ void tc_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}

// Generic-proxy writes to shared memory become visible to the MMA.
__device__ __forceinline__ void fence_async_smem() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// Shared-memory operand descriptor for the 128-byte swizzle (operands sit in
// 1024-byte atoms of 8 rows x 128 bytes):
//   K-major   rows of 64 elements of the summed index; 8-row groups follow
//             each other (stride 1024), the leading offset is not used.
//   MN-major  rows of 64 elements along the tile's side, one row per value of
//             the summed index; 8-row groups are 1024 bytes apart (stride),
//             the next 64 elements along the side 8192 bytes (leading).
template <bool MN>
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr) {
  const uint64_t lead = MN ? 8192u >> 4 : 1u;
  const uint64_t stride = 1024u >> 4;
  return static_cast<uint64_t>((addr & 0x3FFFFu) >> 4) | (lead << 16) |
         (stride << 32) | (1ull << 46) /* sm_100 descriptor */ |
         (2ull << 61) /* 128-byte swizzle */;
}
// 16 further along the summed index, in descriptor units.
template <bool MN>
__device__ __forceinline__ constexpr uint32_t operand_step() {
  return (MN ? 16u * 128u : 32u) >> 4;
}

// Instruction descriptor of kind::f16: f32 accumulators, both operands bf16
// or both f16, M x N.
template <bool A_MN, bool B_MN>
__device__ __forceinline__ uint32_t mma_desc(uint32_t m, uint32_t n,
                                             bool is_f16) {
  const uint32_t type = is_f16 ? 0u : 1u;
  return (1u << 4) | (type << 7) | (type << 10) |
         (static_cast<uint32_t>(A_MN) << 15) |
         (static_cast<uint32_t>(B_MN) << 16) | ((n >> 3) << 17) |
         ((m >> 4) << 24);
}

template <int CG>
__device__ __forceinline__ void mma_f16(uint32_t tmem, uint64_t a, uint64_t b,
                                        uint32_t desc, bool accumulate) {
  if (CG == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(
            tmem),
        "l"(a), "l"(b), "r"(desc), "r"(static_cast<uint32_t>(accumulate))
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(
            tmem),
        "l"(a), "l"(b), "r"(desc), "r"(static_cast<uint32_t>(accumulate))
        : "memory");
}

// `bar` gets one arrival when every MMA this thread issued so far is done.
__device__ __forceinline__ void mma_commit(uint64_t *bar) {
  asm volatile(
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 "
      "[%0];" ::"r"(smem_addr(bar))
      : "memory");
}
// The same barrier in both CTAs of the pair.
__device__ __forceinline__ void mma_commit_pair(uint64_t *bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster."
      "multicast::cluster.b64 [%0], %1;" ::"r"(smem_addr(bar)),
      "h"(static_cast<uint16_t>(3))
      : "memory");
}

// 16 consecutive f32 columns of this warp's 32 lanes.
__device__ __forceinline__ void tmem_load16(uint32_t addr, float (&v)[16]) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]),
        "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i)
    v[i] = __uint_as_float(r[i]);
}

// The shared::cluster address of `p` in CTA `rank` of this cluster.
__device__ __forceinline__ uint32_t cluster_addr(const void *p, uint32_t rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
               : "=r"(remote)
               : "r"(smem_addr(p)), "r"(rank));
  return remote;
}

__device__ __forceinline__ float4 ld_cluster_v4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

__device__ __forceinline__ void mbar_arrive_cluster(uint32_t addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(
                   addr)
               : "memory");
}

// A tile into this CTA's shared memory, its bytes counted on the barrier at
// the shared::cluster address `bar` (the pair's first CTA's).
__device__ __forceinline__ void tma_load_2d_pair(void *dst,
                                                 const CUtensorMap *map,
                                                 int32_t x, int32_t y,
                                                 uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::"
      "complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}

}  // namespace hexir
