// async.cuh — device-side building blocks that every kernel file shares:
// packed f32 arithmetic, programmatic dependent launch, the cluster barrier's
// halves, bounded mbarrier waits and bulk copies.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace nbk {

constexpr unsigned FULL = 0xffffffffu;

// Packed two-lane f32 arithmetic (PTX add/fma .rn.f32x2): each component
// rounded to nearest exactly as the scalar .rn instruction.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
      "add.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rc, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tmov.b64 rc, {%6, %7};\n\t"
      "fma.rn.f32x2 rd, ra, rb, rc;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}

// Programmatic dependent launch. Every kernel of the token loop is launched
// with programmatic stream serialisation: it may start while its predecessor
// on the stream still runs. pdl_wait() blocks until the predecessor grid has
// completed and its writes are visible; pdl_trigger() lets the successor
// start once every CTA of this grid has triggered or exited. Every CTA passes
// pdl_wait() before it triggers or exits, so when a kernel starts, every
// launch before its immediate predecessor has completed. Before pdl_wait() a
// kernel therefore writes nothing to global memory and reads only the
// model's constant weights and data that launches at least two back (or the
// host, before the pass) produced; it reads the latter through L2
// (ld.global.cg), never through a possibly stale L1 line.
__device__ __forceinline__ void pdl_trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// The two halves of a cluster barrier. Distributed shared memory is usable once
// every CTA of the cluster is known to run: an arrive where the kernel starts
// and the wait before its first remote access cost next to nothing.
__device__ __forceinline__ void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }

// Bounded mbarrier waits: a wait that gives up returns false, and its caller
// raises the device error flag and skips the work instead of hanging.
constexpr uint32_t MBAR_WAIT_LIMIT = 1u << 24;

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ bool mbar_wait_polls(uint32_t bar, uint32_t phase, uint32_t polls) {
  for (uint32_t i = 0; i < polls; ++i) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(phase)
        : "memory");
    if (done) return true;
  }
  return false;
}
// The same, given up also once another thread of the block has.
__device__ __forceinline__ bool mbar_wait_polls(uint32_t bar, uint32_t phase, uint32_t polls, const int* failed) {
  for (uint32_t i = 0; i < polls; i += 64) {
    if (mbar_wait_polls(bar, phase, 64)) return true;
    if (*static_cast<const volatile int*>(failed)) return false;
  }
  return false;
}
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t phase) {
  for (uint32_t i = 0; i < MBAR_WAIT_LIMIT; ++i) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(phase)
        : "memory");
    if (done) return true;
  }
  return false;
}

// Bulk copies (cp.async.bulk) of contiguous global ranges into shared memory,
// completing on one mbarrier: one thread initialises the barrier, announces
// the bytes and issues every copy; addresses and sizes are 16-byte multiples.
__device__ __forceinline__ void bulk_start(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(1) : "memory");
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bulk_copy(void* dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src),
               "r"(bytes), "r"(bar)
               : "memory");
}

}  // namespace nbk
