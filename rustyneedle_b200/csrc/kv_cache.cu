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

// The row's scale and its reciprocal step; a row that cannot be held is NaN. A
// row of zeros has the smallest scale: the attention's weights are normalised
// by the largest exponent with the value scale in it, and a row that gives
// nothing must not push those that give something out of f16.
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
__device__ __forceinline__ void load_elements(const T* p, T (&x)[N]) {
  struct alignas(sizeof(T) * N) Pack {
    T v[N];
  };
  const Pack q = *reinterpret_cast<const Pack*>(p);
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = q.v[i];
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

constexpr int ROW_WARPS = 8, ROW_AHEAD = 4;

// Where a row goes: found once for all of the row's units, a unit being the
// keys or the values of one head. Finding it is a chain of four loads from
// far (two steps of the search, the span, the page), about 3 us, against 256
// bytes a unit: with a warp for each unit 24000 rows of 8 heads of 128 took
// 135 us to append and 111 to read, with a warp for a row, 4 units at a time,
// 97 and 70 (59 and 35 by the blocks of 16 rows below: 2.5 and 4.3 TB/s).
struct RowPlace {
  size_t block;  // of head 0 in the pool
  int at;        // position within the page
  bool ok;
};

__device__ __forceinline__ RowPlace place_of(const KvCacheDev& c, const KvBatchDev& b, int row) {
  RowPlace p;
  p.ok = false;
  p.block = 0;
  p.at = 0;
  const int lane = threadIdx.x & 31;
  const int s = sequence_of(b, row);
  const Span sp = span_of(b, s);
  if (!sp.ok) return p;  // check_spans reports it
  if (row < sp.first || row >= sp.first + sp.n) return p;
  const int position = sp.len - sp.n + (row - sp.first);
  const uint32_t page = b.pages[(size_t)s * b.page_stride + position / KV_PAGE];
  if (page >= c.pages) {
    if (lane == 0) atomicOr(c.error, KV_BAD_PAGE);
    return p;
  }
  p.block = (size_t)page * c.kv_heads;
  p.at = position % KV_PAGE;
  p.ok = true;
  return p;
}

// Reports the sequences that break their bounds, wherever their rows lie (a
// sequence behind the batch's rows is met by none of them): a thread for each,
// in blocks behind those that take the rows.
__device__ __forceinline__ void check_spans(const KvCacheDev& c, const KvBatchDev& b, unsigned block) {
  const long long s = (long long)block * (ROW_WARPS * 32) + threadIdx.x;
  if (s < b.sequences && !span_of(b, (int)s).ok) atomicOr(c.error, KV_BAD_SEQUENCE);
}

__global__ void __launch_bounds__(ROW_WARPS * 32) k_kv_check_spans(KvCacheDev c, KvBatchDev b) { check_spans(c, b, blockIdx.x); }

static unsigned span_blocks(const KvBatchDev& b) { return (unsigned)((b.sequences + ROW_WARPS * 32 - 1) / (ROW_WARPS * 32)); }

cudaError_t kv_check_spans(const KvCacheDev& c, const KvBatchDev& b, cudaStream_t st) {
  if (b.sequences == 0) return cudaSuccess;
  k_kv_check_spans<<<span_blocks(b), ROW_WARPS * 32, 0, st>>>(c, b);
  return cudaGetLastError();
}

// A warp for `each` units of a row (a multiple of four, or all that there
// are). grid row_blocks = ceil(rows · shares / 8), and those of check_spans;
// block 256.
template <typename T, int D, bool E4M3>
__global__ void __launch_bounds__(ROW_WARPS * 32) k_kv_append(KvCacheDev c, KvBatchDev b, RowsDev keys, RowsDev values, bool vector, int each, int shares, unsigned row_blocks) {
  if (blockIdx.x >= row_blocks) return check_spans(c, b, blockIdx.x - row_blocks);
  constexpr int N = D / 32;
  const int lane = threadIdx.x & 31;
  const long long item = (long long)blockIdx.x * ROW_WARPS + (threadIdx.x >> 5);
  if (item >= (long long)b.rows * shares) return;
  const int row = (int)(item / shares), u0 = (int)(item % shares) * each, u1 = min(c.kv_heads * 2, u0 + each);
  const RowPlace place = place_of(c, b, row);
  if (!place.ok) return;
  for (int u = u0; u < u1; u += ROW_AHEAD) {
    float x[ROW_AHEAD][N];
#pragma unroll
    for (int i = 0; i < ROW_AHEAD; ++i) {
      if (u + i >= u1) break;
      const RowsDev& in = (u + i) & 1 ? values : keys;
      load_elements<T, N>(static_cast<const T*>(in.data) + row * in.row_stride + ((u + i) >> 1) * in.head_stride + lane * N, vector, x[i]);
    }
#pragma unroll
    for (int i = 0; i < ROW_AHEAD; ++i) {
      if (u + i >= u1) break;
      float peak = 0.0f;
      bool finite = true;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        peak = fmaxf(peak, fabsf(x[i][e]));
        finite = finite && fabsf(x[i][e]) <= KV_PEAK_MAX;
      }
      peak = __uint_as_float(__reduce_max_sync(FULL, __float_as_uint(peak)));
      const RowScale r = row_scale<E4M3>(peak, __all_sync(FULL, finite));
      uint8_t code[N];
#pragma unroll
      for (int e = 0; e < N; ++e) code[e] = !r.held ? 0 : E4M3 ? quantise_e4m3(x[i][e], r) : (uint8_t)(int8_t)quantise_int8(x[i][e], r);
      const size_t block = place.block + ((u + i) >> 1);
      if (!((u + i) & 1)) {
        uint8_t* dst = c.k + block * (KV_PAGE * D) + key_byte(place.at, lane * N);
        if constexpr (N == 2)
          *reinterpret_cast<uint16_t*>(dst) = (uint16_t)(code[0] | code[1] << 8);
        else
          *reinterpret_cast<uint32_t*>(dst) = (uint32_t)code[0] | (uint32_t)code[1] << 8 | (uint32_t)code[2] << 16 | (uint32_t)code[3] << 24;
        if (lane == 0) c.ks[block * KV_PAGE + place.at] = r.scale;
      } else {
        uint8_t* dst = c.v + block * (KV_PAGE * D);
#pragma unroll
        for (int e = 0; e < N; ++e) dst[value_byte(place.at, lane * N + e, D)] = code[e];
        if (lane == 0) c.vs[block * KV_PAGE + place.at] = r.scale;
      }
    }
  }
}

// The same units, read back: code · scale, rounded once.
template <typename T, int D, bool E4M3>
__global__ void __launch_bounds__(ROW_WARPS * 32) k_kv_read(KvCacheDev c, KvBatchDev b, RowsDev keys, RowsDev values, bool vector, int each, int shares, unsigned row_blocks) {
  if (blockIdx.x >= row_blocks) return check_spans(c, b, blockIdx.x - row_blocks);
  constexpr int N = D / 32;
  const int lane = threadIdx.x & 31;
  const long long item = (long long)blockIdx.x * ROW_WARPS + (threadIdx.x >> 5);
  if (item >= (long long)b.rows * shares) return;
  const int row = (int)(item / shares), u0 = (int)(item % shares) * each, u1 = min(c.kv_heads * 2, u0 + each);
  const RowPlace place = place_of(c, b, row);
  if (!place.ok) return;
  for (int u = u0; u < u1; u += ROW_AHEAD) {
    uint8_t code[ROW_AHEAD][N];
    float scale[ROW_AHEAD];
#pragma unroll
    for (int i = 0; i < ROW_AHEAD; ++i) {
      if (u + i >= u1) break;
      const size_t block = place.block + ((u + i) >> 1);
      const bool value = (u + i) & 1;
      scale[i] = (value ? c.vs : c.ks)[block * KV_PAGE + place.at];
      if (!value) {
        load_elements<uint8_t, N>(c.k + block * (KV_PAGE * D) + key_byte(place.at, lane * N), code[i]);
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e) code[i][e] = c.v[block * (KV_PAGE * D) + value_byte(place.at, lane * N + e, D)];
      }
    }
#pragma unroll
    for (int i = 0; i < ROW_AHEAD; ++i) {
      if (u + i >= u1) break;
      float x[N];
#pragma unroll
      for (int e = 0; e < N; ++e) x[e] = __fmul_rn(code_value<E4M3>(code[i][e]), scale[i]);
      const RowsDev& out = (u + i) & 1 ? values : keys;
      store_elements<T, N>(static_cast<T*>(out.data) + row * out.row_stride + ((u + i) >> 1) * out.head_stride + lane * N, vector, x);
    }
  }
}

// Sixteen consecutive rows of one head a warp, for calls whose sequences bring
// that many: their places are found together, and where they follow one
// another in a page, four positions' value codes of a dimension, which the pool
// keeps together, are written (read) as one word.
constexpr int BLOCK_ROWS = 16;

// The places of rows r0 .. r0 + 15, lane i and lane i + 16 holding row r0 + i's:
// one search by the whole warp for the first row, one by each lane behind it
// for rows of later sequences. Returns whether they follow one another in a page.
__device__ __forceinline__ bool block_places(const KvCacheDev& c, const KvBatchDev& b, int r0, RowPlace* place) {
  const int lane = threadIdx.x & 31, row = r0 + (lane & 15);
  RowPlace p;
  p.ok = false;
  p.block = 0;
  p.at = 0;
  int s = sequence_of(b, r0);
  if (row < b.rows) {
    if (b.row_start[s + 1] <= row) {
      int hi = b.sequences;  // row_start[s] <= row: the last such s below hi
      while (hi - s > 1) {
        const int mid = (s + hi) / 2;
        if (b.row_start[mid] <= row)
          s = mid;
        else
          hi = mid;
      }
    }
    const Span sp = span_of(b, s);
    if (sp.ok && row >= sp.first && row < sp.first + sp.n) {
      const int position = sp.len - sp.n + (row - sp.first);
      const uint32_t page = b.pages[(size_t)s * b.page_stride + position / KV_PAGE];
      p.ok = page < c.pages;
      p.block = (size_t)page * c.kv_heads;
      p.at = position % KV_PAGE;
      if (!p.ok) atomicOr(c.error, KV_BAD_PAGE);
    }
  }
  *place = p;
  const unsigned long long first = __shfl_sync(FULL, (unsigned long long)p.block, 0);
  const int at = __shfl_sync(FULL, p.at, 0);
  return __all_sync(FULL, p.ok && p.block == first && p.at == at + (lane & 15));
}

// The scale of a row whose largest magnitude has these bits (a NaN's bits are
// above an infinity's, those above every number's).
template <bool E4M3>
__device__ __forceinline__ RowScale row_scale_of_bits(uint32_t peak) {
  return row_scale<E4M3>(__uint_as_float(peak), peak <= __float_as_uint(KV_PEAK_MAX));
}

// Four numbers as codes in a word.
template <bool E4M3>
__device__ __forceinline__ uint32_t quantise4(const float* x, const RowScale& r) {
  if constexpr (E4M3) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(__fmul_rn(x[1], r.inverse)), "f"(__fmul_rn(x[0], r.inverse)));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(__fmul_rn(x[3], r.inverse)), "f"(__fmul_rn(x[2], r.inverse)));
    return r.held ? (uint32_t)lo | (uint32_t)hi << 16 : 0u;
  } else {
    // quantise_int8's first guess, in the low byte of 1.5 · 2^23 + n; its
    // correction only where a remainder reaches half a scale
    uint32_t bits[4];
    bool near = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float shifted = __fadd_rn(__fmul_rn(x[i], r.inverse), 12582912.0f);
      bits[i] = __float_as_uint(shifted);
      near = near || !(fabsf(__fmaf_rn(-__fadd_rn(shifted, -12582912.0f), r.scale, x[i])) < 0.5f * r.scale);
    }
    if (near) {  // also where the row is not held: its scale is NaN
#pragma unroll
      for (int i = 0; i < 4; ++i) bits[i] = r.held ? (uint32_t)quantise_int8(x[i], r) : 0u;
    }
    return __byte_perm(__byte_perm(bits[0], bits[1], 0x0040), __byte_perm(bits[2], bits[3], 0x0040), 0x5410);
  }
}

template <bool E4M3>
__device__ __forceinline__ void code_values4(uint32_t w, float scale, float (&x)[4]) {
  const uint2 h = widen<E4M3, false>(w);
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&h.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&h.y));
  x[0] = __fmul_rn(a.x, scale);
  x[1] = __fmul_rn(a.y, scale);
  x[2] = __fmul_rn(b.x, scale);
  x[3] = __fmul_rn(b.y, scale);
}

template <int N>
__device__ __forceinline__ uint32_t peak_bits(const float (&x)[N]) {
  uint32_t p = 0;
#pragma unroll
  for (int e = 0; e < N; ++e) p = max(p, __float_as_uint(x[e]) & 0x7fffffffu);
#pragma unroll
  for (int o = 8; o; o >>= 1) p = max(p, __shfl_xor_sync(FULL, p, o));  // a half warp's
  return p;
}

// A half warp a row: lanes 0 - 15 rows 0 - 7, lanes 16 - 31 rows 8 - 15, D / 16
// dimensions a lane. grid row_blocks = ceil(rows / 16 / 8) · kv_heads, the heads of
// the same rows next to one another (they lie side by side in the dense buffers),
// and those of check_spans; block 256.
// Four CTAs an SM (64 registers) rather than three: 32768 int8 rows of 8 heads
// of 128 took 93 us against 117, 24000 e4m3 rows 59.5 against 62.3.
template <typename T, int D, bool E4M3>
__global__ void __launch_bounds__(ROW_WARPS * 32, 4) k_kv_append_block(KvCacheDev c, KvBatchDev b, RowsDev keys, RowsDev values, bool vector16, unsigned row_blocks) {
  if (blockIdx.x >= row_blocks) return check_spans(c, b, blockIdx.x - row_blocks);
  constexpr int M = D / 16, AHEAD = sizeof(T) == 4 && D == 128 ? 1 : 2;
  const int lane = threadIdx.x & 31, h = blockIdx.x % c.kv_heads;
  const long long r0 = ((long long)(blockIdx.x / c.kv_heads) * ROW_WARPS + (threadIdx.x >> 5)) * BLOCK_ROWS;
  if (r0 >= b.rows) return;
  const T* kp = static_cast<const T*>(keys.data) + h * keys.head_stride;
  const T* vp = static_cast<const T*>(values.data) + h * values.head_stride;
  RowPlace place;
  const bool whole = block_places(c, b, (int)r0, &place);
  const int d0 = (lane & 15) * M, upper = lane >> 4;
  uint32_t words[M][2] = {};  // row i of the half's eight is byte i % 4 of [.][i / 4]
  float key_scale = 0.0f, value_scale = 0.0f;  // of row lane % 16
#pragma unroll
  for (int i0 = 0; i0 < 8; i0 += AHEAD) {
    float x[2][AHEAD][M];
    size_t block[AHEAD];
    int at[AHEAD];
    bool ok[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int own = upper * 8 + i0 + i;
      block[i] = __shfl_sync(FULL, (unsigned long long)place.block, own) + h;
      at[i] = __shfl_sync(FULL, place.at, own);
      ok[i] = __shfl_sync(FULL, (int)place.ok, own);
#pragma unroll
      for (int e = 0; e < M; ++e) x[0][i][e] = x[1][i][e] = 0.0f;
      if (ok[i]) {
        load_elements<T, M>(kp + (r0 + own) * keys.row_stride + d0, vector16, x[0][i]);
        load_elements<T, M>(vp + (r0 + own) * values.row_stride + d0, vector16, x[1][i]);
      }
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const RowScale rk = row_scale_of_bits<E4M3>(peak_bits(x[0][i])), rv = row_scale_of_bits<E4M3>(peak_bits(x[1][i]));
      if ((lane & 15) == upper * 8 + i0 + i) key_scale = rk.scale, value_scale = rv.scale;
      uint32_t code[M / 4], value[M / 4];
#pragma unroll
      for (int e = 0; e < M / 4; ++e) {
        code[e] = quantise4<E4M3>(&x[0][i][4 * e], rk);
        value[e] = quantise4<E4M3>(&x[1][i][4 * e], rv);
      }
      if (ok[i]) {
        uint8_t* dst = c.k + block[i] * (KV_PAGE * D) + key_byte(at[i], d0);
        if constexpr (M == 4)
          *reinterpret_cast<uint32_t*>(dst) = code[0];
        else
          *reinterpret_cast<uint2*>(dst) = make_uint2(code[0], code[1]);
        if (!whole) {
#pragma unroll
          for (int e = 0; e < M; ++e) c.v[block[i] * (KV_PAGE * D) + value_byte(at[i], d0 + e, D)] = (uint8_t)(value[e / 4] >> (8 * (e % 4)));
        }
      }
#pragma unroll
      for (int e = 0; e < M; ++e) {  // the code of dimension e into its word's byte
        const int into = (i0 + i) & 3, y = e & 3;
        const uint32_t w = value[e / 4];
        words[e][(i0 + i) >> 2] |= (into >= y ? w << (8 * (into - y)) : w >> (8 * (y - into))) & (0xffu << (8 * into));
      }
    }
  }
  // a row's scale by the lane of its own half
  if ((lane & 15) / 8 == upper && place.ok) {
    c.ks[(place.block + h) * KV_PAGE + place.at] = key_scale;
    c.vs[(place.block + h) * KV_PAGE + place.at] = value_scale;
  }
  if (!whole) return;
  const int first = __shfl_sync(FULL, place.at, 0);
  const size_t block = place.block + h;
  // the pool's word k holds the positions 4 (at / 4 + k) .. + 3, that is, rows 4 k - s ..; the
  // lower half writes words 0 and 1, the upper one 2, 3 and what is left in 4
  const int s = first % 4, quad = first / 4 * 4;
#pragma unroll
  for (int e = 0; e < M; ++e) {
    const uint32_t below = __shfl_xor_sync(FULL, words[e][1], 16);
    uint8_t* dst = c.v + block * (KV_PAGE * D) + value_byte(0, d0 + e, D);
    const uint32_t w0 = __funnelshift_l(upper ? below : 0u, words[e][0], 8 * s), w1 = __funnelshift_l(words[e][0], words[e][1], 8 * s);
    const int at0 = quad + upper * 8;
    uint8_t* p0 = dst + value_byte(at0, 0, D);
    if (upper || s == 0) {
      *reinterpret_cast<uint32_t*>(p0) = w0;
    } else {
#pragma unroll
      for (int byte = 1; byte < 4; ++byte)
        if (byte >= s) p0[byte] = (uint8_t)(w0 >> (8 * byte));
    }
    *reinterpret_cast<uint32_t*>(dst + value_byte(at0 + 4, 0, D)) = w1;
    if (upper && s != 0) {
      const uint32_t w2 = __funnelshift_l(words[e][1], 0u, 8 * s);
      uint8_t* p2 = dst + value_byte(quad + 16, 0, D);
#pragma unroll
      for (int byte = 0; byte < 3; ++byte)
        if (byte < s) p2[byte] = (uint8_t)(w2 >> (8 * byte));
    }
  }
}

template <typename T, int D, bool E4M3>
__global__ void __launch_bounds__(ROW_WARPS * 32) k_kv_read_block(KvCacheDev c, KvBatchDev b, RowsDev keys, RowsDev values, bool vector16, unsigned row_blocks) {
  if (blockIdx.x >= row_blocks) return check_spans(c, b, blockIdx.x - row_blocks);
  constexpr int M = D / 16;
  const int lane = threadIdx.x & 31, h = blockIdx.x % c.kv_heads;
  const long long r0 = ((long long)(blockIdx.x / c.kv_heads) * ROW_WARPS + (threadIdx.x >> 5)) * BLOCK_ROWS;
  if (r0 >= b.rows) return;
  T* kp = static_cast<T*>(keys.data) + h * keys.head_stride;
  T* vp = static_cast<T*>(values.data) + h * values.head_stride;
  RowPlace place;
  const bool whole = block_places(c, b, (int)r0, &place);
  const int d0 = (lane & 15) * M, upper = lane >> 4;
  const float key_scale = place.ok ? c.ks[(place.block + h) * KV_PAGE + place.at] : 0.0f, value_scale = place.ok ? c.vs[(place.block + h) * KV_PAGE + place.at] : 0.0f;
  uint32_t words[M][2] = {};
  if (whole) {
    const int first = __shfl_sync(FULL, place.at, 0), s = first % 4, quad = first / 4 * 4 + upper * 8;
#pragma unroll
    for (int e = 0; e < M; ++e) {
      const uint8_t* src = c.v + (place.block + h) * (KV_PAGE * D) + value_byte(0, d0 + e, D);
      const uint32_t w0 = *reinterpret_cast<const uint32_t*>(src + value_byte(quad, 0, D)), w1 = *reinterpret_cast<const uint32_t*>(src + value_byte(quad + 4, 0, D));
      const uint32_t w2 = s ? *reinterpret_cast<const uint32_t*>(src + value_byte(quad + 8, 0, D)) : 0u;
      words[e][0] = __funnelshift_r(w0, w1, 8 * s);
      words[e][1] = __funnelshift_r(w1, w2, 8 * s);
    }
  }
#pragma unroll
  for (int i0 = 0; i0 < 8; i0 += 4) {
    uint32_t code[4][M / 4], value[4][M / 4];
    bool ok[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int own = upper * 8 + i0 + i;
      const size_t block = __shfl_sync(FULL, (unsigned long long)place.block, own) + h;
      const int at = __shfl_sync(FULL, place.at, own);
      ok[i] = __shfl_sync(FULL, (int)place.ok, own);
#pragma unroll
      for (int e = 0; e < M / 4; ++e) {
        code[i][e] = ok[i] ? *reinterpret_cast<const uint32_t*>(c.k + block * (KV_PAGE * D) + key_byte(at, d0 + 4 * e)) : 0u;
        if (whole) {
          // the row's codes of four dimensions, byte i of their words
          const uint32_t lo = __byte_perm(words[4 * e][i0 / 4], words[4 * e + 1][i0 / 4], 0x0040 + 0x0011 * i);
          const uint32_t hi = __byte_perm(words[4 * e + 2][i0 / 4], words[4 * e + 3][i0 / 4], 0x0040 + 0x0011 * i);
          value[i][e] = __byte_perm(lo, hi, 0x5410);
        } else {
          value[i][e] = 0u;
          if (ok[i]) {
#pragma unroll
            for (int y = 0; y < 4; ++y) value[i][e] |= (uint32_t)c.v[block * (KV_PAGE * D) + value_byte(at, d0 + 4 * e + y, D)] << (8 * y);
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int own = upper * 8 + i0 + i;
      const float ks = __shfl_sync(FULL, key_scale, own), vs = __shfl_sync(FULL, value_scale, own);
      float x[M], y[M];
#pragma unroll
      for (int e = 0; e < M / 4; ++e) {
        float four[4], vals[4];
        code_values4<E4M3>(code[i][e], ks, four);
        code_values4<E4M3>(value[i][e], vs, vals);
#pragma unroll
        for (int k = 0; k < 4; ++k) x[4 * e + k] = four[k], y[4 * e + k] = vals[k];
      }
      if (ok[i]) {
        store_elements<T, M>(kp + (r0 + own) * keys.row_stride + d0, vector16, x);
        store_elements<T, M>(vp + (r0 + own) * values.row_stride + d0, vector16, y);
      }
    }
  }
}

__global__ void k_kv_fill_scales(float* ks, float* vs, size_t n) {
  for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (size_t)gridDim.x * blockDim.x) ks[i] = vs[i] = KV_SCALE_MIN;
}

// A fresh pool holds rows of zeros, at a row of zeros' scale: no code of it is
// ever a NaN.
cudaError_t kv_pool_clear(const KvCacheDev& c, cudaStream_t st) {
  const size_t blocks = (size_t)c.pages * c.kv_heads, bytes = blocks * KV_PAGE * c.dim;
  cudaError_t e = cudaMemsetAsync(c.k, 0, bytes, st);
  if (e == cudaSuccess) e = cudaMemsetAsync(c.v, 0, bytes, st);
  if (e == cudaSuccess) e = cudaMemsetAsync(c.error, 0, sizeof(uint32_t), st);
  if (e != cudaSuccess) return e;
  k_kv_fill_scales<<<1184, 256, 0, st>>>(c.ks, c.vs, blocks * KV_PAGE);
  return cudaGetLastError();
}

// What was reported is taken out of the report word, and no more: kernels of
// another stream may have added to it meanwhile.
__global__ void k_kv_clear_report(uint32_t* error, uint32_t reported) { atomicAnd(error, ~reported); }

cudaError_t kv_clear_report(const KvCacheDev& c, uint32_t reported, cudaStream_t st) {
  k_kv_clear_report<<<1, 1, 0, st>>>(c.error, reported);
  return cudaGetLastError();
}

static bool aligned_rows(const RowsDev& r, int size, int n) {
  return reinterpret_cast<uintptr_t>(r.data) % (size * n) == 0 && r.row_stride % n == 0 && r.head_stride % n == 0;
}

template <typename T, int D, bool E4M3>
static cudaError_t rows_launch(bool append, const KvCacheDev& c, const KvBatchDev& b, const RowsDev& keys, const RowsDev& values, cudaStream_t st) {
  const bool vector = aligned_rows(keys, sizeof(T), D / 32) && aligned_rows(values, sizeof(T), D / 32);
  // Blocks of rows where most of them can lie in one sequence and page, and
  // there are enough of them to fill the SMs. A row a warp against blocks, in us:
  //   one sequence, 4 heads of 64:   4096 rows 8.8 : 10.5 append, 5.5 : 5.4 read; 8192 13.5 : 11.6, 8.7 : 6.0
  //   one sequence, 8 heads of 128:  2048 rows 12.2 : 14.3, 6.8 : 7.3; 4096 21.3 : 17.4, 11.1 : 8.2
  //   32768 rows of 8 heads of 128, sequences of 24: 147 : 102, 91 : 55
  if (b.max_rows >= BLOCK_ROWS && (long long)b.rows * c.kv_heads >= 148 * 16 * BLOCK_ROWS / 2) {
    // a lane's D / 16 elements in accesses of at most 16 bytes
    const bool vector16 = aligned_rows(keys, sizeof(T), D / 16) && aligned_rows(values, sizeof(T), D / 16);
    const unsigned blocks = (unsigned)((b.rows + BLOCK_ROWS * ROW_WARPS - 1) / (BLOCK_ROWS * ROW_WARPS)) * c.kv_heads;
    if (append)
      k_kv_append_block<T, D, E4M3><<<blocks + span_blocks(b), ROW_WARPS * 32, 0, st>>>(c, b, keys, values, vector16, blocks);
    else
      k_kv_read_block<T, D, E4M3><<<blocks + span_blocks(b), ROW_WARPS * 32, 0, st>>>(c, b, keys, values, vector16, blocks);
    return cudaGetLastError();
  }
  // all units of a row for a warp, unless that leaves SMs short of warps (16
  // each): one row of 8 heads of 128 took 9.8 us with all of them and 3.9 with
  // four a warp, 4096 rows of 64 heads 192 and 203.
  const int units = c.kv_heads * 2;
  int each = (units + 3) / 4 * 4;
  while (each > 4 && (long long)b.rows * ((units + each - 1) / each) < 148 * 16) each = (each / 2 + 3) / 4 * 4;
  const int shares = (units + each - 1) / each;
  const unsigned grid = (unsigned)(((long long)b.rows * shares + ROW_WARPS - 1) / ROW_WARPS);
  if (append)
    k_kv_append<T, D, E4M3><<<grid + span_blocks(b), ROW_WARPS * 32, 0, st>>>(c, b, keys, values, vector, each, shares, grid);
  else
    k_kv_read<T, D, E4M3><<<grid + span_blocks(b), ROW_WARPS * 32, 0, st>>>(c, b, keys, values, vector, each, shares, grid);
  return cudaGetLastError();
}

template <typename T>
static cudaError_t rows_launch(bool append, const KvCacheDev& c, const KvBatchDev& b, const RowsDev& keys, const RowsDev& values, cudaStream_t st) {
  if (c.dim == 64)
    return c.e4m3 ? rows_launch<T, 64, true>(append, c, b, keys, values, st) : rows_launch<T, 64, false>(append, c, b, keys, values, st);
  return c.e4m3 ? rows_launch<T, 128, true>(append, c, b, keys, values, st) : rows_launch<T, 128, false>(append, c, b, keys, values, st);
}

static cudaError_t rows_launch(bool append, const KvCacheDev& c, const KvBatchDev& b, const RowsDev& keys, const RowsDev& values, cudaStream_t st) {
  if (b.rows == 0) return kv_check_spans(c, b, st);
  if (b.sequences == 0) return cudaSuccess;
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
