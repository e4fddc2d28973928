// kv_attend_wide.cu — the shared-prefix attention where many query rows meet
// the same keys (the prefix of a batch, the tails of long questions): tiles of
// 128 rows on the tcgen05 tensor cores.
//
// A CTA holds two slots, each an accumulator of 128 rows:
//   two tiles: the slots are two row tiles and share every key tile, so the
//              8-bit codes are widened once for 256 rows;
//   one tile:  the slots are one row tile over alternate key tiles.
// While one slot's scores go through the softmax, the tensor cores work for
// the other. Warps 0-3 and 4-7 are the slots' softmax (a warp has 32 rows),
// warps 8-11 load codes and widen them into shared memory, one lane of warp 12
// issues the matrix instructions:
//   S = Q K^T   Q and K codes (f16 or bf16) from shared memory, f32 in TMEM
//   O += P V    P (f16) from TMEM, over the first half of S; V codes (f16)
//
// The softmax reads TMEM in 16-lane pieces of 256 bits a row, so a thread has
// 4 rows x 32 keys of the tile (rows lane / 4 + 8 k, keys 8 n + 2 (lane % 4)
// and the next), not 1 x 128: a key's numbers (scale, the value scale's
// logarithm and reciprocal) then serve 4 rows of a thread, a quarter of the
// shared-memory reads.
//
// O is rescaled in TMEM only when a row's maximum has grown by more than
// SLACK: until then the weights just get larger, up to 2^(HEADROOM + SLACK).
//
// Per 128 keys and slot: 4 · 128 · 128 · D flops on the tensor cores (512
// cycles at D = 64, 1024 at D = 128) and 16384 exponentials (1024 cycles of the
// special-function units). Measured at 40000 shared keys, 512 rows of 8 kv
// heads, D = 128: 139 us, about 6700 cycles for a key tile of two slots, whose
// matrix instructions take 2048. No single unit is what it waits for: copies
// without the exponentials, the maximum, the weights, the widening, the global
// loads or one of the two products were 0 to 19% faster each, and one without
// all of them still took 65 us, the chain of hand-offs from score to weights to
// product: a slot's product waits for all weights of a tile, its next scores for
// the whole product, and the warps that find the maximum also rescale O. More
// slots would fill it, but two have all of TMEM at D = 128;
// key tiles of 64 with two score buffers a slot were slower (161 us), as were
// an issuing warp for each slot (145) and 16 softmax warps (147).
#include "kv_attend.cuh"

namespace nbk {

constexpr int WIDE_ROWS = 128, WIDE_KEYS = 128, WIDE_ATT_THREADS = 16 * 32;
constexpr int WIDE_LOADERS = 4;  // warps
constexpr float SLACK = 6.0f;

// K-major operands without swizzle: 8 rows x 16 bytes make a core matrix of
// 128 contiguous bytes; `sbo` leads to the next 8 rows, 128 to the next 16 bytes.
__device__ __forceinline__ uint64_t core_desc(uint32_t addr, uint32_t sbo) {
  return (uint64_t)((addr >> 4) & 0x3fff) | ((uint64_t)(128 >> 4) << 16) | ((uint64_t)((sbo >> 4) & 0x3fff) << 32) | (1ull << 46);
}

// The issuing warp runs as a whole, its operands the same in every lane, so
// that they can live in uniform registers, and one elected lane issues: 170 us
// for a call that took 174 with one lane of a diverged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t leader;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(leader));
  return leader != 0;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  if (accumulate)
    asm volatile("tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, 1;" ::"r"(d), "l"(a), "l"(b), "r"(idesc) : "memory");
  else
    asm volatile("tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, 0;" ::"r"(d), "l"(a), "l"(b), "r"(idesc) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  if (accumulate)
    asm volatile("tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, 1;" ::"r"(d), "r"(a), "l"(b), "r"(idesc) : "memory");
  else
    asm volatile("tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, 0;" ::"r"(d), "r"(a), "l"(b), "r"(idesc) : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// One arrival for a warp: a call of long questions took 133 us, with an
// arrival from every lane (several hundred a tile) 141.
__device__ __forceinline__ void warp_arrive(uint32_t bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}

// 128 columns of 16 lanes: registers 4 n, 4 n + 1 are row lane / 4, columns 8 n +
// 2 (lane % 4) and the next; 4 n + 2, 4 n + 3 the same of row lane / 4 + 8.
__device__ __forceinline__ void tmem_load(uint32_t addr, uint32_t (&r)[64]) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]), "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
      : "r"(addr));
}
// 32 columns of 16 lanes: registers 4 n, 4 n + 1 are row lane / 4, columns 8 n +
// 2 (lane % 4) and the next; 4 n + 2, 4 n + 3 the same of row lane / 4 + 8.
__device__ __forceinline__ void tmem_load(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}
// The inverse of the 32-column load.
__device__ __forceinline__ void tmem_store(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// 16 columns of 32 bits of 16 lanes: register 2 n is row lane / 4, column 4 n +
// lane % 4, register 2 n + 1 the same of row lane / 4 + 8: pairs of f16 from the
// 256-bit load's neighbouring columns.
__device__ __forceinline__ void tmem_store(uint32_t addr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.16x128b.x4.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

__device__ __forceinline__ bool wait(uint32_t bar, uint32_t phase) { return mbar_wait_polls(bar, phase, ATTEND_POLLS); }

// The launch's 512 threads hold 128 registers each; the four warpgroups share
// them out anew as 192 + 192 + 88 + 40 = 4 x 128.
template <int N>
__device__ __forceinline__ void registers_up() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void registers_down() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// A thread's 4 x 32 scores to weights 2^(t + base): packed as f16 for the
// product, over the columns of S, and summed over inv. PARTIAL: scores of -inf
// are keys that the row does not see, whose inv may be anything.
constexpr uint32_t HALF_LANES = 16u << 16;  // a warp's lanes 16 .. 31
template <bool PARTIAL>
__device__ __forceinline__ void weigh(const float2 (&t)[4][16], const float2 (&base)[4], const float* inv, uint32_t p_addr, float2 (&l)[4]) {
#pragma unroll
  for (int x0 = 0; x0 < 16; x0 += 4) {
    uint32_t p[2][8];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const float2 in = *reinterpret_cast<const float2*>(inv + 8 * (x0 + x));
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 y = t[k][x0 + x];
        float2 own = in;
        if (PARTIAL) own = make_float2(y.x == -INFINITY ? 0.0f : in.x, y.y == -INFINITY ? 0.0f : in.y);
        float2 w = add2(y, base[k]);
        w = make_float2(ex2(w.x), ex2(w.y));
        l[k] = fma2(w, own, l[k]);
        p[k >> 1][2 * x + (k & 1)] = pack_f16(w.x, w.y);
      }
    }
    tmem_store(p_addr + x0 * 4, p[0]);
    tmem_store(p_addr + HALF_LANES + x0 * 4, p[1]);
  }
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

template <int D>
struct WideSmem {
  uint8_t q[2][WIDE_ROWS * D * 2];   // [slot or 0] rows x D
  uint8_t k[2][WIDE_KEYS * D * 2];   // [stage] keys x D
  uint8_t v[2][D * WIDE_KEYS * 2];   // [stage] D x keys
  // per key, four tiles deep (a tile's numbers live from its K's loading until
  // its P is done; K of tile j is written once S of tile j - 2 is complete)
  float mul[4][WIDE_KEYS], add[4][WIDE_KEYS], inv[4][WIDE_KEYS];
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], done, ended, never;
  uint32_t tmem;
  int failed;
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
      bar_init(smem_u32(&sm.p_full[i]), WIDE_ROWS / 32);
    }
    bar_init(smem_u32(&sm.done), 1);
    bar_init(smem_u32(&sm.ended), 1);
    bar_init(smem_u32(&sm.never), 1);
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
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = sm.tmem;

  // A role whose wait runs out ends, and the others' waits for it run out in
  // their turn; `done` completes only if every product was issued. (A look at
  // sm.failed in every wait ended all of them at once, and took 5 % of the kernel.)
  bool ok = true;
  if (warp < 8) {
    // ------------------------------------------------------------- softmax
    registers_up<192>();
    const int slot = warp >> 2, g = lane >> 2, c2 = (lane & 3) * 2;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem + lanes + slot * 128, o_addr = tmem + lanes + 256 + slot * 128;
    // the thread's rows: first + 8 k
    const int first = row0 + (pair ? slot * WIDE_ROWS : 0) + (warp & 3) * 32 + g;
    int limit[4];  // keys below it are seen by row k
#pragma unroll
    for (int k = 0; k < 4; ++k) limit[k] = prefix ? k1 : min(k1, sees0 + min(first + 8 * k, rows - 1) / a.group + 1);
    // keys below it are seen by every row of the warp
    const int all_see = prefix ? k1 : min(k1, sees0 + min(first - g, rows - 1) / a.group + 1);
    float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    float2 l[4] = {};
    int n = 0;
    for (int e = slot; e < events && ok; e += 2, ++n) {
      const int j = pair ? e >> 1 : e, key0 = k0 + j * WIDE_KEYS;
      ok = __all_sync(FULL, wait(smem_u32(&sm.s_full[slot]), n & 1));
      if (!ok) break;
      fence_after();
      const float* mul = sm.mul[j & 3] + c2;
      const float* add = sm.add[j & 3] + c2;
      const float* inv = sm.inv[j & 3] + c2;
      float2 t[4][16];
      {
        uint32_t lo[64], hi[64];
        tmem_load(s_addr, lo);
        tmem_load(s_addr + HALF_LANES, hi);
        tmem_wait_load();
#pragma unroll
        for (int x = 0; x < 16; ++x) {
          const float2 mu = *reinterpret_cast<const float2*>(mul + 8 * x), ad = *reinterpret_cast<const float2*>(add + 8 * x);
          t[0][x] = fma2(make_float2(__uint_as_float(lo[4 * x]), __uint_as_float(lo[4 * x + 1])), mu, ad);
          t[1][x] = fma2(make_float2(__uint_as_float(lo[4 * x + 2]), __uint_as_float(lo[4 * x + 3])), mu, ad);
          t[2][x] = fma2(make_float2(__uint_as_float(hi[4 * x]), __uint_as_float(hi[4 * x + 1])), mu, ad);
          t[3][x] = fma2(make_float2(__uint_as_float(hi[4 * x + 2]), __uint_as_float(hi[4 * x + 3])), mu, ad);
        }
      }
      const bool partial = key0 + WIDE_KEYS > all_see && !prefix;
      if (partial) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int x = 0; x < 16; ++x) {
            t[k][x].x = key0 + 8 * x + c2 < limit[k] ? t[k][x].x : -INFINITY;
            t[k][x].y = key0 + 8 * x + c2 + 1 < limit[k] ? t[k][x].y : -INFINITY;
          }
      }
      float want[4];
      bool grown = false;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float top = fmaxf(t[k][0].x, t[k][0].y);
#pragma unroll
        for (int x = 1; x < 16; ++x) top = max3(top, t[k][x].x, t[k][x].y);
        top = fmaxf(top, __shfl_xor_sync(FULL, top, 1));
        top = fmaxf(top, __shfl_xor_sync(FULL, top, 2));
        want[k] = __fadd_rn(top, -HEADROOM);
        grown = grown || want[k] > __fadd_rn(m[k], SLACK) || (m[k] == -INFINITY && want[k] != -INFINITY);
      }
      if (__any_sync(FULL, grown)) {
        float keep[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float next = fmaxf(m[k], want[k]);
          keep[k] = next == m[k] ? 1.0f : ex2(__fadd_rn(m[k], -next));
          m[k] = next;
          l[k] = make_float2(__fmul_rn(l[k].x, keep[k]), __fmul_rn(l[k].y, keep[k]));
        }
        if (n > 0) {
#pragma unroll 1
          for (int c = 0; c < 2 * D; c += 32) {  // both halves of the lanes
            const uint32_t at = o_addr + (c % D) + (c < D ? 0u : HALF_LANES);
            const float low = c < D ? keep[0] : keep[2], high = c < D ? keep[1] : keep[3];
            uint32_t o[16];
            tmem_load(at, o);
            tmem_wait_load();
#pragma unroll
            for (int x = 0; x < 16; ++x) o[x] = __float_as_uint(__fmul_rn(__uint_as_float(o[x]), x & 2 ? high : low));
            tmem_store(at, o);
          }
        }
      }
      // weights 2^(t - m): packed as f16 for the product, over columns of S (all
      // of which have been read), and summed over inv
      float2 base[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) base[k].x = base[k].y = m[k] == -INFINITY ? 0.0f : -m[k];
      if (partial)
        weigh<true>(t, base, inv, s_addr, l);
      else
        weigh<false>(t, base, inv, s_addr, l);
      tmem_wait_store();
      fence_before();
      warp_arrive(smem_u32(&sm.p_full[slot]));
    }
    if (!ok) sm.failed = 1;
    if (ok && tiles > 0) ok = __all_sync(FULL, mbar_wait_polls(smem_u32(&sm.done), 0, ATTEND_POLLS, &sm.failed));
    fence_after();
    // the rows' part; a slot without a key tile of its own has sum 0
    if (ok) {
      const int index = parts0 + (pair ? part : 2 * part + slot);
      size_t at[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int r = first + 8 * k;
        at[k] = r < rows ? ((size_t)index * a.b.rows + token0 + r / a.group) * a.heads + h * a.group + r % a.group : 0;
        float sum = __fadd_rn(l[k].x, l[k].y);
        sum = __fadd_rn(sum, __shfl_xor_sync(FULL, sum, 1));
        sum = __fadd_rn(sum, __shfl_xor_sync(FULL, sum, 2));
        if (r < rows && c2 == 0) a.part_ml[at[k]] = make_float2(m[k], sum);
      }
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        uint32_t o[2][16];
        if (n > 0) {
          tmem_load(o_addr + c, o[0]);
          tmem_load(o_addr + HALF_LANES + c, o[1]);
          tmem_wait_load();
        } else {
#pragma unroll
          for (int x = 0; x < 16; ++x) o[0][x] = o[1][x] = 0u;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (first + 8 * k < rows) {
#pragma unroll
            for (int x = 0; x < 4; ++x)
              *reinterpret_cast<uint2*>(a.part_o + at[k] * D + c + 8 * x + c2) = make_uint2(o[k >> 1][4 * x + (k & 1) * 2], o[k >> 1][4 * x + (k & 1) * 2 + 1]);
          }
      }
    } else {
      // no part of these rows: their sum is NaN, and so is what it is joined into
      sm.failed = 1;
      const int index = parts0 + (pair ? part : 2 * part + slot);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int r = first + 8 * k;
        if (r < rows && c2 == 0) a.part_ml[((size_t)index * a.b.rows + token0 + r / a.group) * a.heads + h * a.group + r % a.group] = make_float2(0.0f, NAN);
      }
    }
  } else if (warp < 12) {
    // -------------------------------------------------------------- loading
    // K's registers are loaded for the next tile while V is widened, and V's
    // while the next K is; the page two tiles ahead is known by then.
    registers_down<88>();
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
      if (j >= 2) ok = __all_sync(FULL, wait(smem_u32(&sm.k_empty[stage]), ((j >> 1) - 1) & 1));
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
      warp_arrive(smem_u32(&sm.k_full[stage]));
      fetch_k(j + 1, next);
      if (j >= 2) ok = __all_sync(FULL, wait(smem_u32(&sm.v_empty[stage]), ((j >> 1) - 1) & 1));
      if (!ok) break;
#pragma unroll
      for (int x = 0; x < VN; ++x) {
        const uint32_t w0[4] = {vr[x][0].x, vr[x][0].y, vr[x][0].z, vr[x][0].w}, w1[4] = {vr[x][1].x, vr[x][1].y, vr[x][1].z, vr[x][1].w};
        uint8_t* dst = sm.v[stage] + (lw * 4 + (lane >> 4) * 2 + ((lane >> 3) & 1)) * 128 + (lane & 7) * 16;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const uint2 lo = widen<E4M3, false>(w0[t]), hi = widen<E4M3, false>(w1[t]);
          *reinterpret_cast<uint4*>(dst + (x * 4 + t) * V_SBO) = make_uint4(lo.x, lo.y, hi.x, hi.y);
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      warp_arrive(smem_u32(&sm.v_full[stage]));
      fetch_v(j + 1, next);
      page = next;
      next = after;
    }
    if (!ok) sm.failed = 1;
  } else {
    registers_down<40>();
    if (warp == 12) {
      // ------------------------------------------------ the matrix instructions
      // (all 512 columns are allocated: the TMEM address is 0)
      constexpr uint64_t STAGE = WIDE_KEYS * D * 2 / 16;
      const uint64_t q_desc = core_desc(smem_u32(sm.q[0]), ROW_SBO), k_desc = core_desc(smem_u32(sm.k[0]), ROW_SBO), v_desc = core_desc(smem_u32(sm.v[0]), V_SBO);
      auto scores = [&](int e) {
        const int slot = e & 1, j = pair ? e >> 1 : e, stage = j & 1;
        if (!pair || slot == 0) {
          ok = ok && __all_sync(FULL, wait(smem_u32(&sm.k_full[stage]), (j >> 1) & 1));
          fence_after();
        }
        if (!ok) return;
        const uint64_t qa = q_desc + (pair ? slot * (WIDE_ROWS * D * 2 / 16) : 0), ka = k_desc + stage * STAGE;
        if (elect_one()) {
#pragma unroll
          for (int x = 0; x < D / 16; ++x) mma_ss(slot * 128, qa + x * 16, ka + x * 16, S_IDESC, x > 0);
          mma_commit(smem_u32(&sm.s_full[slot]));
          if (!pair || slot == 1) mma_commit(smem_u32(&sm.k_empty[stage]));
        }
        __syncwarp();
      };
      for (int e = 0; e < 2 && e < events; ++e) scores(e);
      if (expires(a.c)) ok = __all_sync(FULL, mbar_wait_polls(smem_u32(&sm.never), 0, EXPIRE_POLLS));
      for (int e = 0; e < events && ok; ++e) {
        const int slot = e & 1, j = pair ? e >> 1 : e, stage = j & 1;
        ok = __all_sync(FULL, wait(smem_u32(&sm.p_full[slot]), (e >> 1) & 1));
        if (ok && (!pair || slot == 0)) ok = __all_sync(FULL, wait(smem_u32(&sm.v_full[stage]), (j >> 1) & 1));
        if (!ok) break;
        fence_after();
        const uint64_t va = v_desc + stage * STAGE;
        if (elect_one()) {
#pragma unroll
          for (int x = 0; x < WIDE_KEYS / 16; ++x) mma_ts(256 + slot * 128, slot * 128 + x * 8, va + x * 16, O_IDESC, e >= 2 || x > 0);
          if (!pair || slot == 1) mma_commit(smem_u32(&sm.v_empty[stage]));
        }
        __syncwarp();
        if (e + 2 < events) scores(e + 2);
      }
      if (ok && events > 0) {
        if (elect_one()) mma_commit(smem_u32(&sm.done));
      } else if (events > 0) {
        sm.failed = 1;
        if (elect_one()) mma_commit(smem_u32(&sm.ended));
        __syncwarp();
        wait(smem_u32(&sm.ended), 0);  // what was issued ends before the TMEM is freed
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
