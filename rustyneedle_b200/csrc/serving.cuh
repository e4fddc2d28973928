// serving.cuh — device helpers shared by the drafted-decoding kernels.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "async.cuh"
#include "serving.h"

namespace nbk {

// A sequence of a batch. `ok` is false for one that breaks its bounds; it is
// then left out by every kernel.
struct Span {
  int first, n, len;
  bool ok;
};

__device__ __forceinline__ Span span_of(const KvBatchDev& b, int s) {
  Span x;
  x.first = b.row_start[s];
  const int end = b.row_start[s + 1];
  x.len = b.lengths[s];
  x.n = end - x.first;
  x.ok = x.first >= 0 && end >= x.first && end <= b.rows && x.n <= b.max_rows && x.len >= x.n && x.len <= b.max_length &&
         (long long)x.len <= (long long)b.page_stride * KV_PAGE;
  return x;
}

// The last sequence whose first row is at most `row` (a warp's lanes together;
// 32 probes a step, so two steps for 1024 sequences). Sequences without rows
// share their successor's start and are passed over. Whatever row_start holds,
// the result is in [0, sequences); the caller checks the span.
__device__ __forceinline__ int sequence_of(const KvBatchDev& b, int row) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = b.sequences;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32;
    const int at = lo + lane * step;
    const bool below = at < hi && b.row_start[at] <= row;
    const unsigned votes = __ballot_sync(FULL, below);
    const int k = votes ? 31 - __clz(votes) : 0;
    lo += k * step;
    hi = min(hi, lo + step);
  }
  return lo;
}

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) {
  return x;
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) {
  return __float2half_rn(x);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}

// Four 8-bit codes (one word) as two pairs of f16 or bf16, exactly.
//   int8 → f16:  (code + 128) in the low byte of 0x6400 is the half 1152 + code.
//   int8 → bf16: 0x4300 | (code & 0x7f) is 128 + the low seven bits and
//                0x4300 | (code & 0x80) is 128, or 256 when the sign bit is set;
//                their difference is the code.
//   e4m3 → bf16: sign, exponent and mantissa shifted into bf16's places give
//                the value times 2^-120 (subnormals included), 2^(7 - 127).
__device__ __forceinline__ uint32_t sub_f16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t sub_bf16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

template <bool E4M3, bool BF16>
__device__ __forceinline__ uint2 widen(uint32_t w) {
  uint2 r;
  if constexpr (!E4M3 && !BF16) {
    const uint32_t u = w ^ 0x80808080u;
    r.x = sub_f16x2(__byte_perm(u, 0x64646464u, 0x4140), 0x64806480u);
    r.y = sub_f16x2(__byte_perm(u, 0x64646464u, 0x4342), 0x64806480u);
  } else if constexpr (!E4M3 && BF16) {
    const uint32_t a = __byte_perm(w, 0x43434343u, 0x4140), b = __byte_perm(w, 0x43434343u, 0x4342);
    r.x = sub_bf16x2(a & 0xff7fff7fu, a & 0xff80ff80u);
    r.y = sub_bf16x2(b & 0xff7fff7fu, b & 0xff80ff80u);
  } else if constexpr (E4M3 && !BF16) {
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, lo;\n\tcvt.rn.f16x2.e4m3x2 %1, hi;\n\t}"
        : "=r"(r.x), "=r"(r.y)
        : "r"(w));
  } else {
    const uint32_t a = __byte_perm(w, 0u, 0x1404), b = __byte_perm(w, 0u, 0x3424);
    r.x = mul_bf16x2((a & 0x80008000u) | ((a & 0x7f007f00u) >> 4), 0x7b807b80u);
    r.y = mul_bf16x2((b & 0x80008000u) | ((b & 0x7f007f00u) >> 4), 0x7b807b80u);
  }
  return r;
}

// One code's value, exactly.
template <bool E4M3>
__device__ __forceinline__ float code_value(uint8_t code) {
  if constexpr (!E4M3) {
    return (float)(int8_t)code;
  } else {
    const uint2 h = widen<true, false>(code);
    return __half2float(__ushort_as_half((unsigned short)(h.x & 0xffff)));
  }
}

}  // namespace nbk
