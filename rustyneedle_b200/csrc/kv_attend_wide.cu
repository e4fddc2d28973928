// kv_attend_wide.cu — the shared-prefix attention where many query rows meet
// the same keys (the prefix of a batch, the tails of long questions): tiles of
// 128 rows on the tcgen05 tensor cores.
//
// A CTA holds two slots, each an accumulator of 128 rows:
//   two tiles: the slots are two row tiles and share every key tile, so the
//              8-bit codes are widened once for 256 rows;
//   one tile:  the slots are one row tile over alternate key tiles.
// While one slot's scores go through the softmax, the tensor cores work for
// the other. Warps 0-3 and 4-7 are the slots' softmax (a thread is a row:
// TMEM lane = row; a row of 128 scores stays in registers between its maximum
// and its exponentials), warps 8-11 load codes and widen them into shared
// memory, one lane of warp 12 issues the matrix instructions:
//   S = Q K^T   Q and K codes (f16 or bf16) from shared memory, f32 in TMEM
//   O += P V    P (f16) from TMEM, over the first half of S; V codes (f16)
// Two modes, chosen by each CTA from the value scales of its own keys:
//   plain  their ratio is at most 2^PLAIN_BITS: the values enter the product as
//          f16(code · scale / R), R the power of two above the largest scale
//          (2^-12 relative, no subnormals), the weights are the softmax's own,
//          and a key costs the softmax one number, its scale
//   exact  otherwise (and for NaN scales): the codes enter as they are and the
//          value scales through the exponents, as in the 16-row kernel
// A number for each key costs every row's thread 4 bytes of shared-memory
// bandwidth, 1024 of a tile pair's 2048 tensor cycles at D = 128: three of
// them made a tile pair 7000 cycles long, one 4000.
//
// O is rescaled in TMEM only when a row's maximum has grown by more than
// SLACK: until then the weights just get larger, up to 2^(HEADROOM + SLACK).
//
// Per 128 keys and slot: 4 · 128 · 128 · D flops on the tensor cores (512
// cycles at D = 64, 1024 at D = 128), 16384 exponentials (1024 cycles of the
// special-function units), so at D = 64 the exponentials bound the kernel and
// at D = 128 both are even.
#include "kv_attend.cuh"

namespace nbk {

constexpr int WIDE_ROWS = 128, WIDE_KEYS = 128, WIDE_ATT_THREADS = 16 * 32;
constexpr int WIDE_LOADERS = 128;
constexpr float SLACK = 6.0f;

// K-major operands without swizzle: 8 rows x 16 bytes make a core matrix of
// 128 contiguous bytes; `sbo` leads to the next 8 rows, 128 to the next 16 bytes.
__device__ __forceinline__ uint64_t core_desc(uint32_t addr, uint32_t sbo) {
  return (uint64_t)((addr >> 4) & 0x3fff) | ((uint64_t)(128 >> 4) << 16) | ((uint64_t)((sbo >> 4) & 0x3fff) << 32) | (1ull << 46);
}

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}

__device__ __forceinline__ void tmem_load32(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, "
      "%21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
        "=r"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_store32(uint32_t addr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, "
      "%21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]),
      "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr), "r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
      "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Every wait here is for work of microseconds.
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t phase) { return mbar_wait_polls(bar, phase, 1u << 18); }

// The launch's 512 threads hold 128 registers each; the four warpgroups share
// them out anew as 184 + 184 + 104 + 40 = 4 x 128.
template <int N>
__device__ __forceinline__ void registers_up() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void registers_down() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// One row's 128 scores t to weights 2^(t + base): packed as f16 for the
// product and summed, in the exact mode over inv. PARTIAL: scores of -inf are
// keys that the row does not see, whose inv may be anything.
template <bool PLAIN, bool PARTIAL>
__device__ __forceinline__ float weigh(const float2 (&t)[64], float base, const float* inv, uint32_t p_addr) {
  const float2 base2 = make_float2(base, base);
  float2 sum0 = make_float2(0.0f, 0.0f), sum1 = sum0;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    uint32_t p[16];
#pragma unroll
    for (int x = 0; x < 16; x += 2) {
      float2 w0 = t[c * 16 + x], w1 = t[c * 16 + x + 1];
      float4 in = make_float4(1.0f, 1.0f, 1.0f, 1.0f);
      if (!PLAIN) in = *reinterpret_cast<const float4*>(inv + c * 32 + x * 2);
      if (!PLAIN && PARTIAL) {
        in.x = w0.x == -INFINITY ? 0.0f : in.x;
        in.y = w0.y == -INFINITY ? 0.0f : in.y;
        in.z = w1.x == -INFINITY ? 0.0f : in.z;
        in.w = w1.y == -INFINITY ? 0.0f : in.w;
      }
      w0 = add2(w0, base2);
      w1 = add2(w1, base2);
      w0 = make_float2(ex2(w0.x), ex2(w0.y));
      w1 = make_float2(ex2(w1.x), ex2(w1.y));
      if (PLAIN) {
        sum0 = add2(sum0, w0);
        sum1 = add2(sum1, w1);
      } else {
        sum0 = fma2(w0, make_float2(in.x, in.y), sum0);
        sum1 = fma2(w1, make_float2(in.z, in.w), sum1);
      }
      p[x] = pack_f16(w0.x, w0.y);
      p[x + 1] = pack_f16(w1.x, w1.y);
    }
    tmem_store16(p_addr + c * 16, p);
  }
  return __fadd_rn(__fadd_rn(sum0.x, sum1.x), __fadd_rn(sum0.y, sum1.y));
}

constexpr int PLAIN_BITS = 12;

template <int D>
struct WideSmem {
  uint8_t q[2][WIDE_ROWS * D * 2];   // [slot or 0] rows x D
  uint8_t k[2][WIDE_KEYS * D * 2];   // [stage] keys x D
  uint8_t v[2][D * WIDE_KEYS * 2];   // [stage] D x keys
  // per key, four tiles deep (a tile's numbers live from its K's loading until
  // its P is done; K of tile j is written once S of tile j - 2 is complete)
  float mul[4][WIDE_KEYS], add[4][WIDE_KEYS], inv[4][WIDE_KEYS];
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], done;
  uint32_t tmem;
  int failed;
  float scale_most[16], scale_least[16];
};

// grid (row tiles (or pairs) x sequences, kv heads, chunks), block 512
template <int D, bool BF16, bool E4M3>
__global__ void __launch_bounds__(WIDE_ATT_THREADS, 1) k_kv_attend_wide(AttendDev a, bool prefix, bool pair, int parts0) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  WideSmem<D>& sm = *reinterpret_cast<WideSmem<D>*>(smem_raw);
  constexpr uint32_t S_IDESC = (1u << 4) | (BF16 ? (1u << 7) | (1u << 10) : 0u) | ((uint32_t)(WIDE_KEYS >> 3) << 17) | ((uint32_t)(WIDE_ROWS >> 4) << 24);
  constexpr uint32_t O_IDESC = (1u << 4) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(WIDE_ROWS >> 4) << 24);
  constexpr uint32_t ROW_SBO = D / 8 * 128, V_SBO = WIDE_KEYS / 8 * 128;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int h = blockIdx.y, part = blockIdx.z, cover = pair ? 2 * WIDE_ROWS : WIDE_ROWS;

  pdl_trigger();  // a launch that may follow starts as SMs become free; it waits for this one where it joins
  int token0, tokens, row0, k0, k1, sees0 = 0;
  const uint32_t* pages;
  if (prefix) {
    row0 = blockIdx.x * cover;
    token0 = 0;
    tokens = a.b.rows;
    k0 = part * a.prefix_chunk;
    k1 = min(a.prefix, k0 + a.prefix_chunk);
    pages = a.prefix_pages;
  } else {
    const int s = blockIdx.x / a.tiles_per_sequence;
    row0 = (blockIdx.x % a.tiles_per_sequence) * cover;
    const Span sp = span_of(a.b, s);
    if (!sp.ok || row0 >= sp.n * a.group) {
      if (!sp.ok && tid == 0) atomicOr(a.c.error, KV_BAD_SEQUENCE);
      pdl_wait();
      return;
    }
    token0 = sp.first;
    tokens = sp.n;
    sees0 = sp.len - sp.n;
    k0 = part * a.tail_chunk;
    k1 = min(sees0 + min(tokens - 1, (row0 + cover - 1) / a.group) + 1, k0 + a.tail_chunk);
    pages = a.b.pages + (size_t)s * a.b.page_stride;
  }
  const int rows = tokens * a.group;
  const int tiles = max(0, (k1 - k0 + WIDE_KEYS - 1) / WIDE_KEYS);
  // events: (key tile, slot) in the order in which the tensor cores take them
  const int events = pair ? 2 * tiles : tiles;

  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sm.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (tid == 0) {
    sm.failed = 0;
    for (int i = 0; i < 2; ++i) {
      bar_init(smem_u32(&sm.k_full[i]), WIDE_LOADERS);
      bar_init(smem_u32(&sm.v_full[i]), WIDE_LOADERS);
      bar_init(smem_u32(&sm.k_empty[i]), 1);
      bar_init(smem_u32(&sm.v_empty[i]), 1);
      bar_init(smem_u32(&sm.s_full[i]), 1);
      bar_init(smem_u32(&sm.p_full[i]), WIDE_ROWS);
    }
    bar_init(smem_u32(&sm.done), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  // the query rows; rows past the end are zeros
  for (int x = tid; x < cover * (D / 8); x += WIDE_ATT_THREADS) {
    const int i = x / (D / 8), chunk = x % (D / 8), r = row0 + i;
    uint4 w = make_uint4(0, 0, 0, 0);
    if (r < rows) {
      const uint16_t* p = static_cast<const uint16_t*>(a.q.data) + (token0 + r / a.group) * a.q.row_stride + (h * a.group + r % a.group) * a.q.head_stride + chunk * 8;
      if (a.q_vector16) {
        w = *reinterpret_cast<const uint4*>(p);
      } else {
        w.x = p[0] | (uint32_t)p[1] << 16;
        w.y = p[2] | (uint32_t)p[3] << 16;
        w.z = p[4] | (uint32_t)p[5] << 16;
        w.w = p[6] | (uint32_t)p[7] << 16;
      }
    }
    const int t = i & (WIDE_ROWS - 1);
    *reinterpret_cast<uint4*>(sm.q[i / WIDE_ROWS] + (t / 8) * ROW_SBO + chunk * 128 + (t % 8) * 16) = w;
  }
  // the value scales of all keys, a half page a warp at once
  float most = 0.0f, least = INFINITY;
  for (int key0 = k0 + warp * 32; key0 < k1; key0 += WIDE_ATT_THREADS) {
    const uint32_t page = pages[key0 / KV_PAGE];
    if (page >= a.c.pages) {
      least = -1.0f;  // its keys are masked one by one
    } else if (key0 + lane < k1) {
      const float vs = a.c.vs[((size_t)page * a.c.kv_heads + h) * KV_PAGE + key0 % KV_PAGE + lane];
      most = fmaxf(most, vs);
      least = vs == vs ? fminf(least, vs) : -1.0f;  // a NaN
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    most = fmaxf(most, __shfl_xor_sync(FULL, most, o));
    least = fminf(least, __shfl_xor_sync(FULL, least, o));
  }
  if (lane == 0) sm.scale_most[warp] = most, sm.scale_least[warp] = least;
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = sm.tmem;
#pragma unroll
  for (int w = 0; w < 16; ++w) most = fmaxf(most, sm.scale_most[w]), least = fminf(least, sm.scale_least[w]);
  const bool plain = least >= __fmul_rn(most, 1.0f / (1 << PLAIN_BITS)) && most > 0.0f;
  // the power of two at or above the largest scale, and its reciprocal (scales lie in [2^-60, 2^34])
  const float unit = plain ? __uint_as_float((__float_as_uint(most) + 0x7fffffu) & 0x7f800000u) : 1.0f;
  const float per_unit = __uint_as_float(0x7f000000u - __float_as_uint(unit));

  bool ok = true;
  if (warp < 8) {
    // ------------------------------------------------------------- softmax
    registers_up<184>();
    const int slot = warp >> 2;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem + lanes + slot * 128, o_addr = tmem + lanes + 256 + slot * 128;
    const int i = (pair ? slot * WIDE_ROWS : 0) + (warp & 3) * 32 + lane, r = row0 + i;
    const int limit = prefix ? k1 : min(k1, sees0 + min(r, rows - 1) / a.group + 1);
    // keys below it are seen by every row of the warp
    const int all_see = prefix ? k1 : min(k1, sees0 + min(r - lane, rows - 1) / a.group + 1);
    float m = -INFINITY;
    float l = 0.0f;
    int n = 0;
    for (int e = slot; e < events && ok; e += 2, ++n) {
      const int j = pair ? e >> 1 : e, key0 = k0 + j * WIDE_KEYS;
      ok = __all_sync(FULL, wait(smem_u32(&sm.s_full[slot]), n & 1));
      if (!ok) break;
      fence_after();
      const float* mul = sm.mul[j & 3];
      const float* add = sm.add[j & 3];
      const float* inv = sm.inv[j & 3];
      const bool partial = key0 + WIDE_KEYS > all_see;
      float2 t[64];
      {
        uint32_t r0[32], r1[32], r2[32], r3[32];
        tmem_load32(s_addr, r0);
        tmem_load32(s_addr + 32, r1);
        tmem_load32(s_addr + 64, r2);
        tmem_load32(s_addr + 96, r3);
        tmem_wait_load();
#pragma unroll
        for (int x = 0; x < 16; ++x) {
          t[x] = make_float2(__uint_as_float(r0[2 * x]), __uint_as_float(r0[2 * x + 1]));
          t[16 + x] = make_float2(__uint_as_float(r1[2 * x]), __uint_as_float(r1[2 * x + 1]));
          t[32 + x] = make_float2(__uint_as_float(r2[2 * x]), __uint_as_float(r2[2 * x + 1]));
          t[48 + x] = make_float2(__uint_as_float(r3[2 * x]), __uint_as_float(r3[2 * x + 1]));
        }
      }
      float top0 = -INFINITY, top1 = -INFINITY;
      if (plain) {
        const float2 zero = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int x = 0; x < 64; x += 2) {
          const float4 mu = *reinterpret_cast<const float4*>(mul + 2 * x);
          t[x] = fma2(t[x], make_float2(mu.x, mu.y), zero);
          t[x + 1] = fma2(t[x + 1], make_float2(mu.z, mu.w), zero);
        }
      } else {
#pragma unroll
        for (int x = 0; x < 64; x += 2) {
          const float4 mu = *reinterpret_cast<const float4*>(mul + 2 * x), ad = *reinterpret_cast<const float4*>(add + 2 * x);
          t[x] = fma2(t[x], make_float2(mu.x, mu.y), make_float2(ad.x, ad.y));
          t[x + 1] = fma2(t[x + 1], make_float2(mu.z, mu.w), make_float2(ad.z, ad.w));
        }
      }
      if (partial) {
#pragma unroll
        for (int x = 0; x < 64; ++x) {
          t[x].x = key0 + 2 * x < limit ? t[x].x : -INFINITY;
          t[x].y = key0 + 2 * x + 1 < limit ? t[x].y : -INFINITY;
        }
      }
#pragma unroll
      for (int x = 0; x < 64; x += 2) {
        top0 = fmaxf(top0, fmaxf(t[x].x, t[x].y));
        top1 = fmaxf(top1, fmaxf(t[x + 1].x, t[x + 1].y));
      }
      const float want = __fadd_rn(fmaxf(top0, top1), -HEADROOM);
      const bool grown = want > __fadd_rn(m, SLACK) || m == -INFINITY;
      if (__any_sync(FULL, grown)) {
        const float next = grown ? fmaxf(m, want) : m;
        const float keep = next == m ? 1.0f : ex2(__fadd_rn(m, -next));
        m = next;
        l = __fmul_rn(l, keep);
        if (n > 0) {
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            tmem_load32(o_addr + c, o);
            tmem_wait_load();
#pragma unroll
            for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__fmul_rn(__uint_as_float(o[x]), keep));
            tmem_store32(o_addr + c, o);
          }
        }
      }
      const float base = m == -INFINITY ? 0.0f : -m;
      // over columns of S, all of which have been read
      float sum;
      if (plain)
        sum = weigh<true, false>(t, base, inv, s_addr);
      else
        sum = partial ? weigh<false, true>(t, base, inv, s_addr) : weigh<false, false>(t, base, inv, s_addr);
      l = __fadd_rn(l, sum);
      tmem_wait_store();
      fence_before();
      bar_arrive(smem_u32(&sm.p_full[slot]));
    }
    if (!ok) sm.failed = 1;
    if (ok && tiles > 0) ok = __all_sync(FULL, wait(smem_u32(&sm.done), 0));
    fence_after();
    // this row's part; a slot without a key tile of its own has sum 0
    if (ok) {
      const int index = parts0 + (pair ? part : 2 * part + slot);
      const size_t at = r < rows ? ((size_t)index * a.b.rows + token0 + r / a.group) * a.heads + h * a.group + r % a.group : 0;
      if (r < rows) a.part_ml[at] = make_float2(m, l);
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        uint32_t o[32];
        if (n > 0) {
          tmem_load32(o_addr + c, o);
          tmem_wait_load();
        } else {
#pragma unroll
          for (int x = 0; x < 32; ++x) o[x] = 0u;
        }
        if (r < rows) {
#pragma unroll
          for (int x = 0; x < 32; x += 4) *reinterpret_cast<uint4*>(a.part_o + at * D + c + x) = make_uint4(__float_as_uint(__fmul_rn(__uint_as_float(o[x]), unit)), __float_as_uint(__fmul_rn(__uint_as_float(o[x + 1]), unit)),
                           __float_as_uint(__fmul_rn(__uint_as_float(o[x + 2]), unit)), __float_as_uint(__fmul_rn(__uint_as_float(o[x + 3]), unit)));
        }
      }
    }
  } else if (warp < 12) {
    // -------------------------------------------------------------- loading
    // K's registers are loaded for the next tile while V is widened, and V's
    // while the next K is; the page two tiles ahead is known by then.
    registers_down<104>();
    const int lw = warp - 8;
    constexpr int KN = D / 16, VN = D / 32;
    uint4 kr[KN];
    uint4 vr[VN][2];
    float ks = 1.0f, vs = 1.0f;
    auto page_of = [&](int j) -> uint32_t {  // of this warp's 32 keys of tile j
      const int key0 = k0 + j * WIDE_KEYS + lw * 32;
      return j < tiles && key0 < k1 ? pages[key0 / KV_PAGE] : 0xffffffffu;
    };
    auto fetch_k = [&](int j, uint32_t page) {
      if (page < a.c.pages) {
        const size_t block = (size_t)page * a.c.kv_heads + h;
        const int in_page = (k0 + j * WIDE_KEYS + lw * 32) % KV_PAGE;
        const uint8_t* kp = a.c.k + block * (KV_PAGE * D) + in_page * 64 + (lane & 7) * 64 + (lane >> 3) * 16;
        // 8 keys x 4 pieces of 16 codes a load
#pragma unroll
        for (int x = 0; x < KN; ++x) kr[x] = *reinterpret_cast<const uint4*>(kp + (x % (D / 64)) * (KV_PAGE * 64) + (x / (D / 64)) * 8 * 64);
        ks = a.c.ks[block * KV_PAGE + in_page + lane];
        vs = a.c.vs[block * KV_PAGE + in_page + lane];
      } else {
#pragma unroll
        for (int x = 0; x < KN; ++x) kr[x] = make_uint4(0, 0, 0, 0);
      }
    };
    float vs8[8];  // the value scales of the lane's eight keys of V
    auto fetch_v = [&](int j, uint32_t page) {
      if (page < a.c.pages) {
        const size_t block = (size_t)page * a.c.kv_heads + h;
        const int in_page = (k0 + j * WIDE_KEYS + lw * 32) % KV_PAGE;
        // two blocks of 16 keys; of each, eight keys of dimension groups 8t + lane % 8
        const uint8_t* p = a.c.v + block * (KV_PAGE * D) + in_page * D + (lane >> 4) * 16 * D + (lane & 7) * 64 + ((lane >> 3) & 1) * 32;
#pragma unroll
        for (int x = 0; x < VN; ++x) {
          vr[x][0] = *reinterpret_cast<const uint4*>(p + x * 512);
          vr[x][1] = *reinterpret_cast<const uint4*>(p + x * 512 + 16);
        }
        const float4* scales = reinterpret_cast<const float4*>(a.c.vs + block * KV_PAGE + in_page + (lane >> 3) * 8);
        const float4 s0 = scales[0], s1 = scales[1];
        vs8[0] = s0.x, vs8[1] = s0.y, vs8[2] = s0.z, vs8[3] = s0.w, vs8[4] = s1.x, vs8[5] = s1.y, vs8[6] = s1.z, vs8[7] = s1.w;
      } else {
#pragma unroll
        for (int x = 0; x < VN; ++x) vr[x][0] = vr[x][1] = make_uint4(0, 0, 0, 0);
      }
    };
    uint32_t page = page_of(0), next = page_of(1);
    fetch_k(0, page);
    fetch_v(0, page);
    for (int j = 0; j < tiles && ok; ++j) {
      const int stage = j & 1;
      const uint32_t after = page_of(j + 2);
      const int key = lw * 32 + lane;
      if (page >= a.c.pages && lane == 0 && k0 + j * WIDE_KEYS + lw * 32 < k1) atomicOr(a.c.error, KV_BAD_PAGE);
      if (j >= 2) ok = wait(smem_u32(&sm.k_empty[stage]), ((j >> 1) - 1) & 1);
      if (!ok) break;
      const bool seen = page < a.c.pages && k0 + j * WIDE_KEYS + key < k1;
      sm.mul[j & 3][key] = seen ? __fmul_rn(ks, a.scale) : 0.0f;
      sm.add[j & 3][key] = seen ? lg2(vs) : -INFINITY;
      sm.inv[j & 3][key] = seen ? __frcp_rn(vs) : 0.0f;
#pragma unroll
      for (int x = 0; x < KN; ++x) {
        const uint32_t w[4] = {kr[x].x, kr[x].y, kr[x].z, kr[x].w};
        uint8_t* dst = sm.k[stage] + (lw * 4 + x / (D / 64)) * ROW_SBO + ((x % (D / 64)) * 8 + (lane >> 3) * 2) * 128 + (lane & 7) * 16;
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const uint2 lo = widen<E4M3, BF16>(w[2 * y]), hi = widen<E4M3, BF16>(w[2 * y + 1]);
          *reinterpret_cast<uint4*>(dst + y * 128) = make_uint4(lo.x, lo.y, hi.x, hi.y);
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      bar_arrive(smem_u32(&sm.k_full[stage]));
      fetch_k(j + 1, next);
      if (j >= 2) ok = wait(smem_u32(&sm.v_empty[stage]), ((j >> 1) - 1) & 1);
      if (!ok) break;
      // scale / R as the sum of two halves: code · (hi + lo), rounded once
      __half2 hi[4], lo[4];
      if (plain) {
        const int first = k0 + j * WIDE_KEYS + lw * 32 + (lane >> 3) * 8;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float s0 = page < a.c.pages && first + 2 * x < k1 ? __fmul_rn(vs8[2 * x], per_unit) : 0.0f;
          const float s1 = page < a.c.pages && first + 2 * x + 1 < k1 ? __fmul_rn(vs8[2 * x + 1], per_unit) : 0.0f;
          hi[x] = __floats2half2_rn(s0, s1);
          const float2 back = __half22float2(hi[x]);
          lo[x] = __floats2half2_rn(__fadd_rn(s0, -back.x), __fadd_rn(s1, -back.y));
        }
      }
      auto scaled = [&](uint32_t codes, int x) -> uint32_t {
        if (!plain) return codes;
        const __half2 c = *reinterpret_cast<const __half2*>(&codes);
        const __half2 v = __hfma2(c, hi[x], __hmul2(c, lo[x]));
        return *reinterpret_cast<const uint32_t*>(&v);
      };
#pragma unroll
      for (int x = 0; x < VN; ++x) {
        const uint32_t w0[4] = {vr[x][0].x, vr[x][0].y, vr[x][0].z, vr[x][0].w}, w1[4] = {vr[x][1].x, vr[x][1].y, vr[x][1].z, vr[x][1].w};
        uint8_t* dst = sm.v[stage] + (lw * 4 + (lane >> 4) * 2 + ((lane >> 3) & 1)) * 128 + (lane & 7) * 16;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const uint2 c0 = widen<E4M3, false>(w0[t]), c1 = widen<E4M3, false>(w1[t]);
          *reinterpret_cast<uint4*>(dst + (x * 4 + t) * V_SBO) = make_uint4(scaled(c0.x, 0), scaled(c0.y, 1), scaled(c1.x, 2), scaled(c1.y, 3));
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      bar_arrive(smem_u32(&sm.v_full[stage]));
      fetch_v(j + 1, next);
      page = next;
      next = after;
    }
    if (!ok) sm.failed = 1;
  } else {
    registers_down<40>();
    if (warp == 12 && lane == 0 && events > 0) {
      // ------------------------------------------------ the matrix instructions
      const uint32_t q_addr = smem_u32(sm.q[0]);
      auto scores = [&](int e) {
        const int slot = e & 1, j = pair ? e >> 1 : e, stage = j & 1;
        if (!pair || slot == 0) {
          ok = ok && wait(smem_u32(&sm.k_full[stage]), (j >> 1) & 1);
          fence_after();
        }
        if (!ok) return;
        const uint32_t qa = q_addr + (pair ? slot * WIDE_ROWS * D * 2 : 0), ka = smem_u32(sm.k[stage]);
  #pragma unroll
        for (int x = 0; x < D / 16; ++x)
          mma_ss(tmem + slot * 128, core_desc(qa + x * 256, ROW_SBO), core_desc(ka + x * 256, ROW_SBO), S_IDESC, x > 0);
        mma_commit(smem_u32(&sm.s_full[slot]));
        if (!pair || slot == 1) mma_commit(smem_u32(&sm.k_empty[stage]));
      };
      scores(0);
      if (events > 1) scores(1);
      for (int e = 0; e < events && ok; ++e) {
        const int slot = e & 1, j = pair ? e >> 1 : e, stage = j & 1;
        ok = wait(smem_u32(&sm.p_full[slot]), (e >> 1) & 1);
        if (ok && (!pair || slot == 0)) ok = wait(smem_u32(&sm.v_full[stage]), (j >> 1) & 1);
        if (!ok) break;
        fence_after();
        const uint32_t va = smem_u32(sm.v[stage]);
  #pragma unroll
        for (int x = 0; x < WIDE_KEYS / 16; ++x)
          mma_ts(tmem + 256 + slot * 128, tmem + slot * 128 + x * 8, core_desc(va + x * 256, V_SBO), O_IDESC, e >= 2 || x > 0);
        if (!pair || slot == 1) mma_commit(smem_u32(&sm.v_empty[stage]));
        if (e + 2 < events) scores(e + 2);
      }
      mma_commit(smem_u32(&sm.done));
      if (!ok) {
        sm.failed = 1;
        wait(smem_u32(&sm.done), 0);  // what was issued ends before the TMEM is freed
      }
    }
    __syncwarp();
  }
  pdl_wait();  // this launch is complete only after the one before it
  fence_before();
  __syncthreads();
  if (warp == 12) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    if (lane == 0 && *static_cast<volatile int*>(&sm.failed)) atomicOr(a.c.error, KV_WAIT_FAILED);
  }
}

template <int D, bool BF16, bool E4M3>
static cudaError_t wide_launch(const AttendDev& a, bool prefix, int tiles, int chunks, bool dependent, cudaStream_t st) {
  static_assert(sizeof(WideSmem<D>) <= 227 * 1024, "fits an SM's shared memory");
  auto kernel = k_kv_attend_wide<D, BF16, E4M3>;
  // an attribute of the current device's context; setting it is idempotent and cheap beside the launch
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(WideSmem<D>));
  if (e != cudaSuccess) return e;
  const bool pair = prefix ? a.prefix_pair : a.tail_pair;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)tiles, (unsigned)a.c.kv_heads, (unsigned)chunks);
  cfg.blockDim = dim3(WIDE_ATT_THREADS);
  cfg.dynamicSmemBytes = sizeof(WideSmem<D>);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = dependent ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, a, prefix, pair, prefix ? 0 : a.prefix_parts);
}

cudaError_t attend_wide(const AttendDev& a, bool prefix, int tiles, int chunks, bool dependent, cudaStream_t st) {
  const bool bf16 = a.q.dtype == DTYPE_BF16;
  if (a.c.dim == 64) {
    if (bf16) return a.c.e4m3 ? wide_launch<64, true, true>(a, prefix, tiles, chunks, dependent, st) : wide_launch<64, true, false>(a, prefix, tiles, chunks, dependent, st);
    return a.c.e4m3 ? wide_launch<64, false, true>(a, prefix, tiles, chunks, dependent, st) : wide_launch<64, false, false>(a, prefix, tiles, chunks, dependent, st);
  }
  if (bf16) return a.c.e4m3 ? wide_launch<128, true, true>(a, prefix, tiles, chunks, dependent, st) : wide_launch<128, true, false>(a, prefix, tiles, chunks, dependent, st);
  return a.c.e4m3 ? wide_launch<128, false, true>(a, prefix, tiles, chunks, dependent, st) : wide_launch<128, false, false>(a, prefix, tiles, chunks, dependent, st);
}

}  // namespace nbk
