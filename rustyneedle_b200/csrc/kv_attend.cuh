// kv_attend.cuh — what the kernels of the shared-prefix attention share.
#pragma once

#include "serving.cuh"

namespace nbk {

constexpr float HEADROOM = 8.0f;

// Every wait here is for work of microseconds; a poll that finds nothing takes
// 4 us, so one gives up after a quarter of a second. That ends its block, whose
// rows become NaN, and the report word says so.
constexpr uint32_t ATTEND_POLLS = 1u << 16, EXPIRE_POLLS = 1u << 10;
__device__ __forceinline__ bool expires(const KvCacheDev& c) { return c.expire && blockIdx.x + blockIdx.y + blockIdx.z == 0; }
constexpr float LOG2E = 1.4426950408889634f;

struct AttendDev {
  KvCacheDev c;
  KvBatchDev b;
  const uint32_t* prefix_pages;
  int prefix, heads, group;
  float scale;  // softmax scale · log2 e
  RowsDev q, out;
  bool q_vector, q_vector16, out_vector;  // rows may be read 8 (16), written 8 bytes at a time
  float* part_o;  // [parts][rows][heads][dim], unnormalised
  float2* part_ml;  // [parts][rows][heads]: maximum (less HEADROOM) and sum
  int prefix_parts, tail_parts;  // parts of a row
  int prefix_chunk, tail_chunk;  // keys of a chunk, multiples of 32 (of 128 for the wide kernel)
  int tiles_per_sequence;
  bool prefix_pair, tail_pair;  // the wide kernel with two row tiles a CTA
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}

// The kernel for many rows (kv_attend_wide.cu) over the prefix or the tails:
// `tiles` 128-row tiles, or pairs of them, times kv_heads times chunks CTAs.
// `dependent`: it follows another launch of the same call.
cudaError_t attend_wide(const AttendDev& a, bool prefix, int tiles, int chunks, bool dependent, cudaStream_t st);

}  // namespace nbk
