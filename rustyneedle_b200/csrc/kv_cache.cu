// kv_cache.cu — rows into and out of the paged 8-bit key/value cache.
//
// A row x of one head becomes 8-bit codes and one f32 scale:
//   int8  scale = fl(peak · fl(1/127)), code = x / scale to the nearest integer, halves to even
//   e4m3  scale = the smallest power of two s with peak ≤ 448 s, code = e4m3(x / s)
// Both are the exact results: a quotient next to the middle between two codes
// falls on its own side (see quantise_int8), and a power of two makes the e4m3
// quotient exact, which costs no accuracy above e4m3's smallest exponent.
#include "serving.cuh"

namespace nbk {

// The row's scale and its reciprocal step; a row that cannot be held is NaN.
struct RowScale {
  float scale, inverse;
  bool held;
};

template <bool E4M3>
__device__ __forceinline__ RowScale row_scale(float peak, bool finite) {
  RowScale r;
  r.held = finite && peak <= KV_PEAK_MAX;
  if (!r.held) {
    r.scale = __int_as_float(0x7fc00000);
    r.inverse = 0.0f;
    return r;
  }
  if (peak == 0.0f) {
    r.scale = r.inverse = 1.0f;
    return r;
  }
  if constexpr (E4M3) {
    // peak = m · 2^e with m in [1, 2); 448 = 1.75 · 2^8
    const uint32_t bits = __float_as_uint(peak);
    int e = (int)(bits >> 23) - 127;
    e += (bits & 0x7fffffu) > 0x600000u ? -7 : -8;
    if (bits < 0x00800000u) e = -200;
    e = max(-60, e);
    r.scale = __uint_as_float((uint32_t)(e + 127) << 23);
    r.inverse = __uint_as_float((uint32_t)(127 - e) << 23);
  } else {
    r.scale = fmaxf(__fmul_rn(peak, 1.0f / 127.0f), KV_SCALE_MIN);
    r.inverse = __frcp_rn(r.scale);
  }
  return r;
}

// x / scale to the nearest integer, halves to even, exactly. The product with
// the rounded reciprocal is within 2^-16 of the quotient, so its nearest
// integer n is the quotient's or its neighbour across a half. x - n · scale is
// then exact in f32 (a multiple of the smaller operand's last bit and at most
// a scale in size), and comparing it with half a scale decides.
__device__ __forceinline__ int quantise_int8(float x, const RowScale& r) {
  const float n = rintf(__fmul_rn(x, r.inverse));
  const float left = __fmaf_rn(-n, r.scale, x), half = 0.5f * r.scale;
  int code = (int)n;
  if (left > half || (left == half && (code & 1))) ++code;
  if (left < -half || (left == -half && (code & 1))) --code;
  return max(-127, min(127, code));
}

__device__ __forceinline__ uint8_t quantise_e4m3(float x, const RowScale& r) {
  uint16_t two;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(two) : "f"(0.0f), "f"(__fmul_rn(x, r.inverse)));
  return (uint8_t)(two & 0xff);
}

// N consecutive elements; one load when the host found them aligned.
template <typename T, int N>
__device__ __forceinline__ void load_elements(const T* p, bool vector, float (&x)[N]) {
  struct alignas(sizeof(T) * N) Pack {
    T v[N];
  };
  if (vector) {
    const Pack q = *reinterpret_cast<const Pack*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = to_f32(q.v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = to_f32(p[i]);
  }
}

template <typename T, int N>
__device__ __forceinline__ void store_elements(T* p, bool vector, const float (&x)[N]) {
  struct alignas(sizeof(T) * N) Pack {
    T v[N];
  };
  if (vector) {
    Pack q;
#pragma unroll
    for (int i = 0; i < N; ++i) q.v[i] = from_f32<T>(x[i]);
    *reinterpret_cast<Pack*>(p) = q;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = from_f32<T>(x[i]);
  }
}

constexpr int ROW_WARPS = 8;

// One warp for each (row, kv head, keys or values). grid ceil(rows · kv_heads
// · 2 / 8), block 256.
template <typename T, int D, bool E4M3>
__global__ void __launch_bounds__(ROW_WARPS * 32) k_kv_append(KvCacheDev c, KvBatchDev b, RowsDev keys, RowsDev values, bool vector) {
  constexpr int N = D / 32;
  const int lane = threadIdx.x & 31;
  const long long unit = (long long)blockIdx.x * ROW_WARPS + (threadIdx.x >> 5);
  if (unit >= (long long)b.rows * c.kv_heads * 2) return;
  const bool value = unit & 1;
  const int h = (int)((unit >> 1) % c.kv_heads), row = (int)((unit >> 1) / c.kv_heads);
  const int s = sequence_of(b, row);
  const Span sp = span_of(b, s);
  if (!sp.ok) {
    if (lane == 0) atomicOr(c.error, KV_BAD_SEQUENCE);
    return;
  }
  if (row < sp.first || row >= sp.first + sp.n) return;
  const int p = sp.len - sp.n + (row - sp.first);
  const uint32_t page = b.pages[(size_t)s * b.page_stride + p / KV_PAGE];
  if (page >= c.pages) {
    if (lane == 0) atomicOr(c.error, KV_BAD_PAGE);
    return;
  }
  const RowsDev& in = value ? values : keys;
  float x[N];
  load_elements<T, N>(static_cast<const T*>(in.data) + row * in.row_stride + h * in.head_stride + lane * N, vector, x);
  float peak = 0.0f;
  bool finite = true;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    peak = fmaxf(peak, fabsf(x[i]));
    finite = finite && fabsf(x[i]) <= KV_PEAK_MAX;
  }
  peak = __uint_as_float(__reduce_max_sync(FULL, __float_as_uint(peak)));
  const RowScale r = row_scale<E4M3>(peak, __all_sync(FULL, finite));
  uint8_t code[N];
#pragma unroll
  for (int i = 0; i < N; ++i) code[i] = !r.held ? 0 : E4M3 ? quantise_e4m3(x[i], r) : (uint8_t)(int8_t)quantise_int8(x[i], r);
  const int at = p % KV_PAGE;
  const size_t block = (size_t)page * c.kv_heads + h;
  if (!value) {
    uint8_t* dst = c.k + block * (KV_PAGE * D) + key_byte(at, lane * N);
    if constexpr (N == 2)
      *reinterpret_cast<uint16_t*>(dst) = (uint16_t)(code[0] | code[1] << 8);
    else
      *reinterpret_cast<uint32_t*>(dst) = (uint32_t)code[0] | (uint32_t)code[1] << 8 | (uint32_t)code[2] << 16 | (uint32_t)code[3] << 24;
    if (lane == 0) c.ks[block * KV_PAGE + at] = r.scale;
  } else {
    uint8_t* dst = c.v + block * (KV_PAGE * D);
#pragma unroll
    for (int i = 0; i < N; ++i) dst[value_byte(at, lane * N + i, D)] = code[i];
    if (lane == 0) c.vs[block * KV_PAGE + at] = r.scale;
  }
}

// The same units, read back: code · scale, rounded once.
template <typename T, int D, bool E4M3>
__global__ void __launch_bounds__(ROW_WARPS * 32) k_kv_read(KvCacheDev c, KvBatchDev b, RowsDev keys, RowsDev values, bool vector) {
  constexpr int N = D / 32;
  const int lane = threadIdx.x & 31;
  const long long unit = (long long)blockIdx.x * ROW_WARPS + (threadIdx.x >> 5);
  if (unit >= (long long)b.rows * c.kv_heads * 2) return;
  const bool value = unit & 1;
  const int h = (int)((unit >> 1) % c.kv_heads), row = (int)((unit >> 1) / c.kv_heads);
  const int s = sequence_of(b, row);
  const Span sp = span_of(b, s);
  if (!sp.ok) {
    if (lane == 0) atomicOr(c.error, KV_BAD_SEQUENCE);
    return;
  }
  if (row < sp.first || row >= sp.first + sp.n) return;
  const int p = sp.len - sp.n + (row - sp.first);
  const uint32_t page = b.pages[(size_t)s * b.page_stride + p / KV_PAGE];
  if (page >= c.pages) {
    if (lane == 0) atomicOr(c.error, KV_BAD_PAGE);
    return;
  }
  const int at = p % KV_PAGE;
  const size_t block = (size_t)page * c.kv_heads + h;
  float x[N];
  if (!value) {
    const uint8_t* src = c.k + block * (KV_PAGE * D) + key_byte(at, lane * N);
    const float scale = c.ks[block * KV_PAGE + at];
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = __fmul_rn(code_value<E4M3>(src[i]), scale);
  } else {
    const uint8_t* src = c.v + block * (KV_PAGE * D);
    const float scale = c.vs[block * KV_PAGE + at];
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = __fmul_rn(code_value<E4M3>(src[value_byte(at, lane * N + i, D)]), scale);
  }
  const RowsDev& out = value ? values : keys;
  store_elements<T, N>(static_cast<T*>(out.data) + row * out.row_stride + h * out.head_stride + lane * N, vector, x);
}

__global__ void k_kv_fill_scales(float* ks, float* vs, size_t n) {
  for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (size_t)gridDim.x * blockDim.x) ks[i] = vs[i] = 1.0f;
}

// A fresh pool holds rows of zeros: no code of it is ever a NaN.
cudaError_t kv_pool_clear(const KvCacheDev& c, cudaStream_t st) {
  const size_t blocks = (size_t)c.pages * c.kv_heads, bytes = blocks * KV_PAGE * c.dim;
  cudaError_t e = cudaMemsetAsync(c.k, 0, bytes, st);
  if (e == cudaSuccess) e = cudaMemsetAsync(c.v, 0, bytes, st);
  if (e == cudaSuccess) e = cudaMemsetAsync(c.error, 0, sizeof(uint32_t), st);
  if (e != cudaSuccess) return e;
  k_kv_fill_scales<<<1184, 256, 0, st>>>(c.ks, c.vs, blocks * KV_PAGE);
  return cudaGetLastError();
}

static bool aligned_rows(const RowsDev& r, int size, int n) {
  return reinterpret_cast<uintptr_t>(r.data) % (size * n) == 0 && r.row_stride % n == 0 && r.head_stride % n == 0;
}

template <typename T, int D, bool E4M3>
static cudaError_t rows_launch(bool append, const KvCacheDev& c, const KvBatchDev& b, const RowsDev& keys, const RowsDev& values, cudaStream_t st) {
  const bool vector = aligned_rows(keys, sizeof(T), D / 32) && aligned_rows(values, sizeof(T), D / 32);
  const long long units = (long long)b.rows * c.kv_heads * 2;
  const unsigned grid = (unsigned)((units + ROW_WARPS - 1) / ROW_WARPS);
  if (append)
    k_kv_append<T, D, E4M3><<<grid, ROW_WARPS * 32, 0, st>>>(c, b, keys, values, vector);
  else
    k_kv_read<T, D, E4M3><<<grid, ROW_WARPS * 32, 0, st>>>(c, b, keys, values, vector);
  return cudaGetLastError();
}

template <typename T>
static cudaError_t rows_launch(bool append, const KvCacheDev& c, const KvBatchDev& b, const RowsDev& keys, const RowsDev& values, cudaStream_t st) {
  if (c.dim == 64)
    return c.e4m3 ? rows_launch<T, 64, true>(append, c, b, keys, values, st) : rows_launch<T, 64, false>(append, c, b, keys, values, st);
  return c.e4m3 ? rows_launch<T, 128, true>(append, c, b, keys, values, st) : rows_launch<T, 128, false>(append, c, b, keys, values, st);
}

static cudaError_t rows_launch(bool append, const KvCacheDev& c, const KvBatchDev& b, const RowsDev& keys, const RowsDev& values, cudaStream_t st) {
  if (b.sequences == 0 || b.rows == 0) return cudaSuccess;
  if (keys.dtype == DTYPE_F32) return rows_launch<float>(append, c, b, keys, values, st);
  if (keys.dtype == DTYPE_F16) return rows_launch<__half>(append, c, b, keys, values, st);
  return rows_launch<__nv_bfloat16>(append, c, b, keys, values, st);
}

cudaError_t kv_append(const KvCacheDev& c, const KvBatchDev& b, const RowsDev& keys, const RowsDev& values, cudaStream_t st) {
  return rows_launch(true, c, b, keys, values, st);
}
cudaError_t kv_read(const KvCacheDev& c, const KvBatchDev& b, const RowsDev& keys, const RowsDev& values, cudaStream_t st) {
  return rows_launch(false, c, b, keys, values, st);
}

}  // namespace nbk
