// kv_attend.cu — attention of a batch over one shared prefix and over each
// sequence's own tail, on the 8-bit paged cache.
//
// With K_j = ks_j · kc_j and V_j = vs_j · vc_j (codes kc, vc; f32 scales ks, vs)
//   t_j = (q·kc_j) · ks_j · scale · log2 e + log2 vs_j      w_j = 2^(t_j - m)
//   out = Σ w_j vc_j / Σ w_j / vs_j
// so the codes enter both products exactly and every scale stays in f32: the
// value scale is folded into the exponent, and dividing it out again gives the
// softmax's own sum. m is the running maximum of t less HEADROOM, so w_j ≤
// 2^HEADROOM; the product with the codes takes w as f16 (2^-11 relative down
// to 2^-14, absolute 2^-25 below), the sums take it as f32. So the largest p_j
// vs_j sets the weights' unit: rows of zeros have the smallest scale (a row of
// zeros of scale 1 with a score 14 above others of 0.02 put 18 % on the result,
// with one 25 above nothing was left of it).
#include <algorithm>
#include <cmath>

#include "kv_attend.cuh"

namespace nbk {

template <bool BF16>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 16 query rows of one kv head against a chunk of the prefix (PREFIX) or of a
// sequence's tail. A row is (token, query head of the group): row r of a tile
// list stands for token r / group. Four warps take the chunk's keys 32 at a
// time in turn and are joined at the end.
//
// The codes come by bulk copies into a ring of ATT_STAGES x 32 keys for each
// warp (one lane asks for them, two groups ahead): 2 D + 8 bytes a key, and
// the kernel is to be bound by those bytes. At D = 64 four CTAs an SM hold 140
// KB in flight.
//
// Lanes: g = lane / 4, c = lane % 4. The key fragment of a 16 x 8 x 16 product
// wants, of key "n = g", four dimensions of the lane's own choice for every
// step, as long as the query fragment has the same: lane c takes 16
// consecutive bytes of every 64, four steps of four dimensions, so a key's
// codes arrive as one 16-byte load. Product j of a block of 16 keys takes the
// keys 4·(n / 2) + 2·j + n % 2, which leaves lane c the scores of the keys 4c
// .. 4c + 3: the order in which the second product wants its left operand, and
// in which the pool keeps the values (value_byte).
constexpr int ATT_WARPS = 4, ATT_STAGES = 2;

template <int D>
struct AttStage {
  uint8_t k[32 * D];  // [D / 64][32][64]
  uint8_t v[32 * D];
  float ks[32], vs[32];
};
template <int D>
struct AttSmem {
  union {
    AttStage<D> ring[ATT_WARPS][ATT_STAGES];
    float o[ATT_WARPS][16][D + 4];  // once every copy has landed and been used
  };
  float2 ml[ATT_WARPS][16];
  uint64_t full[ATT_WARPS][ATT_STAGES], never;
  int failed;
};

template <bool BF16>
__device__ __forceinline__ void store_out4(const RowsDev& out, bool vector, long long at, const float (&y)[4]) {
  uint2 w;
  if constexpr (BF16) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(y[0], y[1]), b = __floats2bfloat162_rn(y[2], y[3]);
    w = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
  } else {
    w = make_uint2(pack_f16(y[0], y[1]), pack_f16(y[2], y[3]));
  }
  uint16_t* p = static_cast<uint16_t*>(out.data) + at;
  if (vector) {
    *reinterpret_cast<uint2*>(p) = w;
  } else {
    p[0] = (uint16_t)w.x;
    p[1] = (uint16_t)(w.x >> 16);
    p[2] = (uint16_t)w.y;
    p[3] = (uint16_t)(w.y >> 16);
  }
}

// A row's running sum: y = Σ w code and sum = Σ w / vs under the maximum top.
struct Joined {
  float top = -INFINITY, sum = 0.0f, y[4] = {};

  // four parts at a time, whose loads are in flight together
  __device__ __forceinline__ void add(const float2 (&ml)[4], const float4 (&v)[4]) {
    const float next = fmaxf(fmaxf(fmaxf(top, ml[0].x), fmaxf(ml[1].x, ml[2].x)), ml[3].x), base = next == -INFINITY ? 0.0f : next;
    const float keep = ex2(__fadd_rn(top, -base));
    top = next;
    sum = __fmul_rn(sum, keep);
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = __fmul_rn(y[e], keep);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float f = ex2(__fadd_rn(ml[i].x, -base));
      sum = __fmaf_rn(ml[i].y, f, sum);
      y[0] = __fmaf_rn(v[i].x, f, y[0]);
      y[1] = __fmaf_rn(v[i].y, f, y[1]);
      y[2] = __fmaf_rn(v[i].z, f, y[2]);
      y[3] = __fmaf_rn(v[i].w, f, y[3]);
    }
  }
  // the parts first, first + step .. of unit (token, head), dimensions d .. d + 3
  template <int D>
  __device__ __forceinline__ void add_parts(const AttendDev& a, size_t stride, size_t unit, int d, int first, int step, int parts) {
    for (int p = first; p < parts; p += 4 * step) {
      float2 ml[4];
      float4 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool some = p + i * step < parts;
        const size_t at = (size_t)(p + i * step) * stride + unit;
        ml[i] = some ? __ldcg(&a.part_ml[at]) : make_float2(-INFINITY, 0.0f);
        v[i] = some ? __ldcg(reinterpret_cast<const float4*>(a.part_o + at * D + d)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      }
      add(ml, v);
    }
  }
  // the attention's values; a row without a key has zeros
  __device__ __forceinline__ void finish() {
    const float norm = sum == 0.0f ? 0.0f : __frcp_rn(sum);
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = __fmul_rn(y[e], norm);
  }
};

// FUSED (tails of one part): the prefix's parts are joined in, and the rows
// written out. Three blocks an SM at D = 128, which is what their rings allow.
template <int D, bool BF16, bool E4M3, bool PREFIX>
__global__ void __launch_bounds__(ATT_WARPS * 32, D == 64 ? 4 : 3) k_kv_attend(AttendDev a, bool fused) {
  constexpr int SEG = D / 64, STEPS = D / 16, NT = D / 8;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  AttSmem<D>& sm = *reinterpret_cast<AttSmem<D>*>(smem_raw);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const int h = blockIdx.y, part = blockIdx.z;
  if (PREFIX) pdl_trigger();
  int token0, tokens, row0, k0, k1, sees0 = 0;  // the tile's rows row0.. of `tokens` tokens from token0; keys [k0, k1)
  const uint32_t* pages;
  if constexpr (PREFIX) {
    row0 = blockIdx.x * 16;
    token0 = 0;
    tokens = a.b.rows;
    k0 = part * a.prefix_chunk;
    k1 = min(a.prefix, k0 + a.prefix_chunk);
    pages = a.prefix_pages;
  } else {
    const int s = blockIdx.x / a.tiles_per_sequence;
    row0 = (blockIdx.x % a.tiles_per_sequence) * 16;
    const Span sp = span_of(a.b, s);
    if (!sp.ok || row0 >= sp.n * a.group) {
      if (!sp.ok && threadIdx.x == 0) atomicOr(a.c.error, KV_BAD_SEQUENCE);
      pdl_wait();
      return;
    }
    token0 = sp.first;
    tokens = sp.n;
    sees0 = sp.len - sp.n;
    k0 = part * a.tail_chunk;
    k1 = min(sees0 + min(tokens - 1, (row0 + 15) / a.group) + 1, k0 + a.tail_chunk);
    pages = a.b.pages + (size_t)s * a.b.page_stride;
  }
  const int rows = tokens * a.group;
  // this warp's groups of 32 keys: k0 + 32 (warp + 4 i), i < count
  const int groups = max(0, (k1 - k0 + 31) / 32), count = max(0, (groups - warp + ATT_WARPS - 1) / ATT_WARPS);
  if (lane == 0)
    for (int i = 0; i < ATT_STAGES; ++i) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_u32(&sm.full[warp][i])) : "memory");
  if (threadIdx.x == 0) {
    sm.failed = 0;
    if (a.c.expire) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_u32(&sm.never)) : "memory");
  }
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  // the pages of the next 32 groups, one a lane
  uint32_t held = 0;
  int held_from = -32;
  auto page_of = [&](int i) {  // by all lanes, with the same i
    if (i >= held_from + 32) {
      held_from = i;
      held = i + lane < count ? pages[(k0 + 32 * (warp + ATT_WARPS * (i + lane))) / KV_PAGE] : 0;
    }
    return __shfl_sync(FULL, held, i - held_from);
  };
  uint32_t bad = 0;  // bit i % 32: group i's page is outside the pool
  auto ask = [&](int i) {
    const uint32_t page = page_of(i);
    const bool ok = page < a.c.pages;
    bad = (bad & ~(1u << (i & 31))) | (ok ? 0u : 1u << (i & 31));
    if (lane == 0) {
      AttStage<D>& st = sm.ring[warp][i % ATT_STAGES];
      const uint32_t bar = smem_u32(&sm.full[warp][i % ATT_STAGES]);
      if (ok) {
        const size_t block = (size_t)page * a.c.kv_heads + h;
        const int in_page = (k0 + 32 * (warp + ATT_WARPS * i)) % KV_PAGE;
        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(64 * D + 256) : "memory");
#pragma unroll
        for (int seg = 0; seg < SEG; ++seg)
          bulk_copy(st.k + seg * 2048, a.c.k + block * (KV_PAGE * D) + seg * (KV_PAGE * 64) + in_page * 64, 2048, bar);
        bulk_copy(st.v, a.c.v + block * (KV_PAGE * D) + in_page * D, 32 * D, bar);
        bulk_copy(st.ks, a.c.ks + block * KV_PAGE + in_page, 128, bar);
        bulk_copy(st.vs, a.c.vs + block * KV_PAGE + in_page, 128, bar);
      } else {
        atomicOr(a.c.error, KV_BAD_PAGE);
        asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
      }
    }
  };
  __syncwarp();
  for (int i = 0; i < min(count, ATT_STAGES); ++i) ask(i);

  // the lane's query fragments; rows past the end are zeros
  uint32_t qf[STEPS][4];
  int limit[2];  // keys below it are seen by rows g and g + 8
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int r = row0 + g + 8 * half;
    const bool live = r < rows;
    const int token = live ? r / a.group : 0;
    limit[half] = PREFIX ? k1 : min(k1, sees0 + token + 1);
    const uint16_t* src = static_cast<const uint16_t*>(a.q.data) + (token0 + token) * a.q.row_stride +
                          (h * a.group + (live ? r % a.group : 0)) * a.q.head_stride;
#pragma unroll
    for (int seg = 0; seg < SEG; ++seg)
#pragma unroll
      for (int st = 0; st < 4; ++st) {
        uint2 x = make_uint2(0, 0);
        if (live) {
          const uint16_t* p = src + seg * 64 + c * 16 + st * 4;
          if (a.q_vector) {
            x = *reinterpret_cast<const uint2*>(p);
          } else {
            x.x = p[0] | (uint32_t)p[1] << 16;
            x.y = p[2] | (uint32_t)p[3] << 16;
          }
        }
        qf[seg * 4 + st][half] = x.x;
        qf[seg * 4 + st][2 + half] = x.y;
      }
  }

  // the tile's upper 8 rows hold something; without them half the softmax is left out
  const bool upper = rows - row0 > 8;
  float o[NT][4] = {};
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
  bool fine = true;
  const int done = count > 0 && warp == 0 && expires(a.c) ? count - 1 : count;  // a test's wait runs out before the last group
  int i = 0;
  for (; i < done; ++i) {
    const int kb = k0 + 32 * (warp + ATT_WARPS * i);
    fine = __all_sync(FULL, mbar_wait_polls(smem_u32(&sm.full[warp][i % ATT_STAGES]), (i / ATT_STAGES) & 1, ATTEND_POLLS));
    if (!fine) break;
    const AttStage<D>& stage = sm.ring[warp][i % ATT_STAGES];
    if (!(bad >> (i & 31) & 1)) {
      float t[2][2][4];  // [block of 16 keys][product][row g: two keys, row g + 8: two keys]
      float inv[2][4];   // 1 / vs of the keys 4c .. 4c + 3
#pragma unroll
      for (int blk = 0; blk < 2; ++blk) {
        const float4 ks = *reinterpret_cast<const float4*>(stage.ks + blk * 16 + c * 4);
        const float4 vs = *reinterpret_cast<const float4*>(stage.vs + blk * 16 + c * 4);
        const float kscale[4] = {ks.x, ks.y, ks.z, ks.w}, vscale[4] = {vs.x, vs.y, vs.z, vs.w};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float s[4] = {};
          const uint8_t* row = stage.k + (blk * 16 + 4 * (g >> 1) + 2 * j + (g & 1)) * 64 + c * 16;
#pragma unroll
          for (int seg = 0; seg < SEG; ++seg) {
            const uint4 w = *reinterpret_cast<const uint4*>(row + seg * 2048);
            const uint32_t word[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int st = 0; st < 4; ++st) {
              const uint2 kf = widen<E4M3, BF16>(word[st]);
              mma16816<BF16>(s, qf[seg * 4 + st], kf.x, kf.y);
            }
          }
#pragma unroll
          for (int e2 = 0; e2 < 2; ++e2) {
            const int e = 2 * j + e2, key = kb + blk * 16 + 4 * c + e;
            const float mul = __fmul_rn(kscale[e], a.scale), add = lg2(vscale[e]);
            inv[blk][e] = key < k1 ? rcp_fast(vscale[e]) : 0.0f;
            // a key that a row does not see gets -inf by selection, whatever lies there
            t[blk][j][e2] = key < limit[0] ? __fmaf_rn(s[e2], mul, add) : -INFINITY;
            if (upper) t[blk][j][2 + e2] = key < limit[1] ? __fmaf_rn(s[2 + e2], mul, add) : -INFINITY;
          }
        }
      }
      float base[2];
      bool grown = false;
      float next[2];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        if (half && !upper) break;
        float top = -INFINITY;
#pragma unroll
        for (int blk = 0; blk < 2; ++blk)
#pragma unroll
          for (int j = 0; j < 2; ++j) top = fmaxf(top, fmaxf(t[blk][j][2 * half], t[blk][j][2 * half + 1]));
        top = fmaxf(top, __shfl_xor_sync(FULL, top, 1));
        top = fmaxf(top, __shfl_xor_sync(FULL, top, 2));
        next[half] = fmaxf(m[half], __fadd_rn(top, -HEADROOM));
        grown = grown || next[half] != m[half];
        base[half] = next[half] == -INFINITY ? 0.0f : next[half];
      }
      if (__any_sync(FULL, grown)) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          if (half && !upper) break;
          const float keep = ex2(__fadd_rn(m[half], -base[half]));  // 0 while nothing was seen
          m[half] = next[half];
          l[half] = __fmul_rn(l[half], keep);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            o[n][2 * half] = __fmul_rn(o[n][2 * half], keep);
            o[n][2 * half + 1] = __fmul_rn(o[n][2 * half + 1], keep);
          }
        }
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        if (half && !upper) break;
#pragma unroll
        for (int blk = 0; blk < 2; ++blk)
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e2 = 0; e2 < 2; ++e2) {
              float& x = t[blk][j][2 * half + e2];
              const bool seen = x != -INFINITY;
              x = ex2(__fadd_rn(x, -base[half]));
              l[half] = seen ? __fmaf_rn(x, inv[blk][2 * j + e2], l[half]) : l[half];
            }
      }
#pragma unroll
      for (int blk = 0; blk < 2; ++blk) {
        const uint32_t pf[4] = {pack_f16(t[blk][0][0], t[blk][0][1]), upper ? pack_f16(t[blk][0][2], t[blk][0][3]) : 0u, pack_f16(t[blk][1][0], t[blk][1][1]),
                                upper ? pack_f16(t[blk][1][2], t[blk][1][3]) : 0u};
#pragma unroll
        for (int tq = 0; tq < D / 32; ++tq) {
          const uint4 w = *reinterpret_cast<const uint4*>(stage.v + blk * 16 * D + tq * 512 + lane * 16);
          const uint32_t word[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const uint2 vf = widen<E4M3, false>(word[n]);
            mma16816<false>(o[tq * 4 + n], pf, vf.x, vf.y);
          }
        }
      }
    }
    __syncwarp();
    if (i + ATT_STAGES < count) ask(i + ATT_STAGES);
  }
  if (done < count) fine = __all_sync(FULL, mbar_wait_polls(smem_u32(&sm.never), 0, EXPIRE_POLLS));
  if (!fine && lane == 0) {  // what was asked for, group i and those behind it, lands before the block ends
    sm.failed = 1;
    atomicOr(a.c.error, KV_WAIT_FAILED);
    for (int j = i; j < min(count, i + ATT_STAGES); ++j) mbar_wait_polls(smem_u32(&sm.full[warp][j % ATT_STAGES]), (j / ATT_STAGES) & 1, ATTEND_POLLS);
  }

  // join the four warps, the ring's memory holding their accumulators
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    l[half] = __fadd_rn(l[half], __shfl_xor_sync(FULL, l[half], 1));
    l[half] = __fadd_rn(l[half], __shfl_xor_sync(FULL, l[half], 2));
    if (c == 0) sm.ml[warp][g + 8 * half] = make_float2(m[half], l[half]);
  }
  __syncthreads();
#pragma unroll
  for (int half = 0; half < 2; ++half)
#pragma unroll
    for (int n = 0; n < NT; ++n) *reinterpret_cast<float2*>(&sm.o[warp][g + 8 * half][n * 8 + 2 * c]) = make_float2(o[n][2 * half], o[n][2 * half + 1]);
  pdl_wait();  // the prefix's parts are complete (and whatever the launch before wrote)
  __syncthreads();
  const int index = PREFIX ? part : a.prefix_parts + part;
  const size_t stride = (size_t)a.b.rows * a.heads;
  for (int x = threadIdx.x; x < 16 * D / 4; x += ATT_WARPS * 32) {
    const int r = x / (D / 4), d = x % (D / 4) * 4;
    if (row0 + r >= rows) break;
    const size_t unit = (size_t)(token0 + (row0 + r) / a.group) * a.heads + h * a.group + (row0 + r) % a.group;
    static_assert(ATT_WARPS == 4, "one step of the sum");
    Joined sum;
    float2 ml[4];
    float4 v[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      ml[w] = sm.ml[w][r];
      v[w] = *reinterpret_cast<const float4*>(&sm.o[w][r][d]);
    }
    sum.add(ml, v);
    if (sm.failed) sum.sum = NAN;  // and so is what it is joined into
    if (!fused) {
      const size_t at = index * stride + unit;
      *reinterpret_cast<float4*>(a.part_o + at * D + d) = make_float4(sum.y[0], sum.y[1], sum.y[2], sum.y[3]);
      if (d == 0) a.part_ml[at] = make_float2(sum.top, sum.sum);
      continue;
    }
    sum.add_parts<D>(a, stride, unit, d, 0, 1, a.prefix_parts);
    sum.finish();
    const int row = token0 + (row0 + r) / a.group, head = h * a.group + (row0 + r) % a.group;
    store_out4<BF16>(a.out, a.out_vector, row * a.out.row_stride + head * a.out.head_stride + d, sum.y);
  }
}

// Joins the parts of a (token, head): D / 4 lanes for each, or for each of
// `ways` shares of its parts, which are then joined in their order. One lane
// group over 128 parts took 19 us of a 37 us call (one row of 16384 keys);
// shares of four parts and more, with four parts' loads in flight, 3 us.
template <int D, bool BF16>
__global__ void __launch_bounds__(256) k_kv_join(AttendDev a, int ways) {
  constexpr int LANES = D / 4, SLOTS = 256 / LANES;
  __shared__ float4 share_o[SLOTS][LANES];
  __shared__ float2 share_ml[SLOTS];
  pdl_wait();
  const int lane = threadIdx.x % LANES, slot = threadIdx.x / LANES, way = slot % ways;
  const long long unit = (long long)blockIdx.x * (SLOTS / ways) + slot / ways;
  const bool some = unit < (long long)a.b.rows * a.heads;
  const int row = some ? (int)(unit / a.heads) : 0, head = some ? (int)(unit % a.heads) : 0;
  // all of a warp's units are of the first one's row or of rows behind it: search for each row that occurs
  int s = 0;
  for (unsigned left = __ballot_sync(FULL, true); left;) {
    const int one = __shfl_sync(FULL, row, __ffs(left) - 1);
    const int found = sequence_of(a.b, one);
    if (row == one) s = found;
    left &= ~__ballot_sync(FULL, row == one);
  }
  const Span sp = span_of(a.b, s);
  const bool live = some && sp.ok && row >= sp.first && row < sp.first + sp.n;
  const int parts = live ? a.prefix_parts + a.tail_parts : 0;
  const size_t stride = (size_t)a.b.rows * a.heads;
  Joined sum;
  sum.add_parts<D>(a, stride, (size_t)unit, lane * 4, way, ways, parts);
  if (ways > 1) {
    share_o[slot][lane] = make_float4(sum.y[0], sum.y[1], sum.y[2], sum.y[3]);
    if (lane == 0) share_ml[slot] = make_float2(sum.top, sum.sum);
    __syncthreads();
    if (way) return;
    for (int w = 1; w < ways; w += 4) {
      float2 ml[4];
      float4 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool some = w + i < ways;
        ml[i] = some ? share_ml[slot + w + i] : make_float2(-INFINITY, 0.0f);
        v[i] = some ? share_o[slot + w + i][lane] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      }
      sum.add(ml, v);
    }
  }
  if (!live) return;
  sum.finish();
  store_out4<BF16>(a.out, a.out_vector, row * a.out.row_stride + head * a.out.head_stride + lane * 4, sum.y);
}

// How a side (the prefix or the tails) is cut: the kernel, its row tiles and
// its chunks of keys. The same plan sizes the workspace.
//
// The plan is the cheapest of all cuts by an estimate in microseconds, whose
// constants were fitted to both kernels, forced, over 2 to 1024 rows, 256 to
// 16384 keys and 4 to 1024 lists (4 kv heads):
//   16 rows:  a CTA's turns (32 keys for each of its four warps) at 1.0 (D = 64)
//             or 1.4 us, and the codes of all tiles at 4.6 TB/s, as the root of
//             the sum of squares
//   128 rows: rounds of one CTA an SM, each 3.5 us and a key tile's time: 1.35
//             or 1.7 us, for two row tiles 2.85 at either width
//   a part:   0.1 us, and its bytes twice at 4 TB/s; the join's launch: 4 us
// Both sides, in us for the call at 4 kv heads, 16 against 128 rows:
//   1024 shared keys, 64 / 128 rows      D = 64  8.1 / 8.9 against 11.0 / 11.9
//   16384 shared keys, 64 / 128 rows     D = 128 34 / 54 against 27 / 30
//   32 sequences of 1024, 16 / 64 rows   D = 64  15 / 26 against 20 / 21
//   32 sequences of 8192, 16 / 64 rows   D = 128 94 / 244 against 144 / 149
// and one against two row tiles of 128:
//   16 sequences of 4096, 256 rows       57 against 59 (D = 64), 82 against 71 (D = 128)
//   16384 shared keys, 256 / 1024 rows   D = 128 40 / 104 against 44 / 97
constexpr double PLAN_PART = 0.1, PLAN_JOIN = 4.0;

// Up to this many parts of the prefix are joined by the tails' own CTAs, more
// by the join's launch. 512 and 2048 shared keys for one row (4 and 16 parts):
// 5.1 and 6.5 us against 7.1 and 7.3; 32768 keys for 5 rows: 20.5 against 15.7.
constexpr int FUSED_PARTS = 16;

struct SidePlan {
  bool wide = false, pair = false;
  int tiles = 0;   // row tiles (prefix: of the batch, tails: of a sequence)
  int chunks = 0;  // of keys
  int chunk = 32, parts = 0;
};

// rows: query rows (token, head of the group) that meet the same `keys`;
// `lists`: how many such sets there are (kv heads, times sequences).
static SidePlan side_plan(long long rows, int keys, long long lists, int dim, bool tail, size_t part_bytes) {
  SidePlan best;
  best.tiles = (int)((rows + 15) / 16);
  if (keys == 0 || lists == 0 || rows == 0) return best;
  double best_us = 0;
  // a part is written and read again, and joined in its turn
  const double part_us = PLAN_PART + part_bytes * 2 / 4e6;
  auto take = [&](double us, bool wide, bool pair, int tiles, int units, int chunks) {
    if (best.chunks && us >= best_us) return;
    best_us = us;
    const int unit = wide ? 128 : 32, each = (units + chunks - 1) / chunks;
    best.wide = wide;
    best.pair = pair;
    best.tiles = tiles;
    best.chunk = each * unit;
    best.chunks = (units + each - 1) / each;
    best.parts = best.chunks * (wide && !pair ? 2 : 1);
  };
  const int groups = (keys + 31) / 32, units = (keys + 127) / 128;
  const long long narrow = (rows + 15) / 16;
  const double bytes_us = (double)lists * narrow * keys * (2 * dim) / 4.6e6;
  for (int n = 1; n <= groups && n <= 64 && (n == 1 || n * part_us < best_us); ++n) {
    const double turns = ((groups + n - 1) / n + ATT_WARPS - 1) / ATT_WARPS * (dim == 64 ? 1.0 : 1.4);
    take(std::sqrt(turns * turns + bytes_us * bytes_us) + n * part_us + (tail && n == 1 ? 0.0 : PLAN_JOIN), false, false, (int)narrow, groups, n);
  }
  for (int pair = 0; pair < (rows > 128 ? 2 : 1); ++pair) {
    const long long tiles = (rows + (pair ? 255 : 127)) / (pair ? 256 : 128);
    const double tile_us = pair ? 2.85 : dim == 64 ? 1.35 : 1.7;
    for (int n = 1; n <= units && n <= 64 && n * part_us < best_us; ++n) {
      const long long rounds = (lists * tiles * n + 147) / 148;
      take((double)rounds * ((units + n - 1) / n * tile_us + 3.5) + n * (pair ? 1 : 2) * part_us + PLAN_JOIN, true, pair, (int)tiles, units, n);
    }
  }
  return best;
}

struct AttendPlan {
  SidePlan prefix, tail;
};

static AttendPlan attend_plan(const KvCacheDev& c, const KvBatchDev& b, int prefix, int heads) {
  const long long group = heads / c.kv_heads;
  const size_t part_bytes = (size_t)b.rows * heads * c.dim * sizeof(float);
  AttendPlan p;
  p.prefix = side_plan(b.rows * group, prefix, c.kv_heads, c.dim, false, part_bytes);
  // also for bounds of no rows or no positions: the tails' kernel reports the sequences that break them
  p.tail = side_plan(std::max(b.max_rows, 1) * group, std::max(b.max_length, 1), (long long)b.sequences * c.kv_heads, c.dim, true, part_bytes);
  return p;
}

size_t kv_attend_workspace(const KvCacheDev& c, const KvBatchDev& b, int prefix, int heads) {
  const AttendPlan p = attend_plan(c, b, prefix, heads);
  const size_t units = (size_t)(p.prefix.parts + p.tail.parts) * b.rows * heads;
  return units * (c.dim * sizeof(float) + sizeof(float2)) + 16;
}

template <typename... P, typename... A>
static cudaError_t launch(void (*kernel)(P...), dim3 grid, int threads, size_t smem, bool dependent, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = dependent ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// The first launch waits for all before it on the stream (the keys and queries
// may just have been written). The ones behind it start early: they read
// nothing of their predecessor before pdl_wait(), and a launch completes only
// after its own pdl_wait(), so the last one finds every part.
template <int D, bool BF16, bool E4M3>
static cudaError_t attend_launch(const AttendDev& d, const AttendPlan& p, cudaStream_t st) {
  constexpr int SMEM = (int)sizeof(AttSmem<D>);
  cudaError_t e = cudaFuncSetAttribute(k_kv_attend<D, BF16, E4M3, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(k_kv_attend<D, BF16, E4M3, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
  bool before = false;  // a launch of this call goes before
  if (e == cudaSuccess && p.prefix.chunks) {
    if (p.prefix.wide)
      e = attend_wide(d, true, p.prefix.tiles, p.prefix.chunks, false, st);
    else
      e = launch(k_kv_attend<D, BF16, E4M3, true>, dim3(p.prefix.tiles, d.c.kv_heads, p.prefix.chunks), ATT_WARPS * 32, SMEM, false, st, d, false);
    before = true;
  }
  bool fused = false;
  if (e == cudaSuccess && p.tail.chunks) {
    const unsigned tiles = (unsigned)d.b.sequences * p.tail.tiles;
    fused = !p.tail.wide && p.tail.parts == 1 && p.prefix.parts <= FUSED_PARTS;
    if (p.tail.wide)
      e = attend_wide(d, false, (int)tiles, p.tail.chunks, before, st);
    else
      e = launch(k_kv_attend<D, BF16, E4M3, false>, dim3(tiles, d.c.kv_heads, p.tail.chunks), ATT_WARPS * 32, SMEM, before, st, d, fused);
    before = true;
  }
  if (e == cudaSuccess && !fused) {
    constexpr int SLOTS = 256 / (D / 4);
    const long long units = (long long)d.b.rows * d.heads;
    int ways = 1;
    while (ways < SLOTS && (d.prefix_parts + d.tail_parts) >= 8 * ways && units * ways < 148 * 4 * SLOTS) ways *= 2;
    const int each = SLOTS / ways;  // units a block
    e = launch(k_kv_join<D, BF16>, dim3((unsigned)((units + each - 1) / each)), 256, 0, before, st, d, ways);
  }
  return e;
}

cudaError_t kv_attend(const KvCacheDev& c, const KvBatchDev& b, const KvAttend& x, cudaStream_t st) {
  if (b.rows == 0) return kv_check_spans(c, b, st);
  if (b.sequences == 0) return cudaSuccess;
  const AttendPlan p = attend_plan(c, b, x.prefix, x.heads);
  AttendDev d;
  d.c = c;
  d.b = b;
  d.prefix_pages = x.prefix_pages;
  d.prefix = x.prefix;
  d.heads = x.heads;
  d.group = x.heads / c.kv_heads;
  d.scale = x.scale * LOG2E;
  d.q = x.query;
  d.out = x.out;
  d.q_vector = reinterpret_cast<uintptr_t>(x.query.data) % 8 == 0 && x.query.row_stride % 4 == 0 && x.query.head_stride % 4 == 0;
  d.q_vector16 = reinterpret_cast<uintptr_t>(x.query.data) % 16 == 0 && x.query.row_stride % 8 == 0 && x.query.head_stride % 8 == 0;
  d.out_vector = reinterpret_cast<uintptr_t>(x.out.data) % 8 == 0 && x.out.row_stride % 4 == 0 && x.out.head_stride % 4 == 0;
  d.prefix_parts = p.prefix.parts;
  d.prefix_chunk = p.prefix.chunk;
  d.prefix_pair = p.prefix.pair;
  d.tail_parts = p.tail.parts;
  d.tail_chunk = p.tail.chunk;
  d.tail_pair = p.tail.pair;
  d.tiles_per_sequence = p.tail.tiles;
  const size_t units = (size_t)(p.prefix.parts + p.tail.parts) * b.rows * x.heads;
  d.part_o = static_cast<float*>(x.workspace);
  d.part_ml = reinterpret_cast<float2*>(d.part_o + units * c.dim);
  const bool bf16 = x.query.dtype == DTYPE_BF16;
  if (c.dim == 64) {
    if (bf16) return c.e4m3 ? attend_launch<64, true, true>(d, p, st) : attend_launch<64, true, false>(d, p, st);
    return c.e4m3 ? attend_launch<64, false, true>(d, p, st) : attend_launch<64, false, false>(d, p, st);
  }
  if (bf16) return c.e4m3 ? attend_launch<128, true, true>(d, p, st) : attend_launch<128, true, false>(d, p, st);
  return c.e4m3 ? attend_launch<128, false, true>(d, p, st) : attend_launch<128, false, false>(d, p, st);
}

}  // namespace nbk
