// verify.cu — drafted tokens against the target's probabilities.
//
// Row i of a sequence has p_i = softmax(x_i / T) over its allowed ids. Draft d
// is accepted while u_i · q_i(d) < p_i(d); at the first rejection the token is
// the lowest id whose running sum of max(p - q, 0) passes u · total, behind the
// last draft the same with p alone. The rows up to the first rejection are
// needed, those behind it are not read (but for a round's, below).
//
// One cluster of CTAs takes a sequence. A round takes `at_once` rows, each
// with its share of the warps: every CTA reads its slice of the vocabulary in
// 16-byte pieces, a thread keeps a running maximum and sum (f32 exponentials;
// joined in f64), every warp's pair goes to every CTA of the cluster, and all
// come to the same decision. The one row that a token is drawn from is read
// once or twice more, from L2, with exponentials and running sums in f64: f32
// sums over a large vocabulary would put some draws on the wrong side of a
// border.
#include <cooperative_groups.h>

#include <cfloat>

#include "serving.cuh"

namespace nbk {

namespace cg = cooperative_groups;

constexpr int VERIFY_THREADS = 512, VERIFY_WARPS = VERIFY_THREADS / 32, VERIFY_MAX_CLUSTER = 8, VERIFY_MAX_ROWS = 8;
constexpr uint32_t NO_TOKEN = 0xffffffffu;

// A logit as the formulas take it: NaN counts as -inf (fmaxf drops it), +inf
// as the largest f32.
__device__ __forceinline__ float tame(float x) { return fminf(fmaxf(x, -INFINITY), FLT_MAX); }

// One row, in pieces of 16 bytes: piece 0 is what lies before the first
// 16-byte boundary, the last one what is left behind the last.
template <typename T>
struct LogitRow {
  static constexpr int N = 16 / sizeof(T);
  const T* p;
  const uint32_t* allowed;  // or null: all ids
  int vocab, head;

  __device__ __forceinline__ LogitRow(const T* row, const uint32_t* mask, int v) : p(row), allowed(mask), vocab(v) {
    head = min(v, (int)((16 - reinterpret_cast<uintptr_t>(row) % 16) % 16 / sizeof(T)));
  }
  // the same for every row of a launch: pieces that any alignment needs
  __device__ __forceinline__ static int pieces(int v) { return v / N + 2; }
  __device__ __forceinline__ int start(int piece) const { return head + (piece - 1) * N; }
  __device__ __forceinline__ bool whole(int piece) const { return start(piece) >= 0 && start(piece) + N <= vocab; }
  __device__ __forceinline__ bool permits(int id) const { return !allowed || (allowed[id >> 5] >> (id & 31) & 1); }
  // which of a piece's ids exist and are allowed
  __device__ __forceinline__ uint32_t live(int piece) const {
    const int e = start(piece);
    uint32_t bits = (1u << N) - 1;
    if (!whole(piece)) {
      if (e < 0) bits &= ~0u << -e;
      if (e + N > vocab) bits &= e >= vocab ? 0u : (1u << (vocab - e)) - 1;
    }
    if (allowed && bits) {
      uint32_t m = 0;
      const int first = max(e, 0), at = first & 31;
      m = allowed[first >> 5] >> at;
      const int last = min(vocab, e + N) - 1;
      if (last >> 5 != first >> 5) m |= allowed[last >> 5] << (32 - at);
      bits &= e < 0 ? m << -e : m;
    }
    return bits;
  }
  __device__ __forceinline__ uint4 raw(int piece) const {
    uint4 w = make_uint4(0, 0, 0, 0);
    const int e = start(piece);
    if (whole(piece)) {
      w = *reinterpret_cast<const uint4*>(p + e);
    } else {
      T x[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        x[i] = from_f32<T>(0.0f);
        if (e + i >= 0 && e + i < vocab) x[i] = p[e + i];
      }
      memcpy(&w, x, 16);
    }
    return w;
  }
  __device__ __forceinline__ static void widen_piece(const uint4& w, float (&x)[N]) {
    T t[N];
    memcpy(t, &w, 16);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = to_f32(t[i]);
  }
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 2^(y / 64) for y <= 0 in f64: y = k + f, k whole, |f| <= 1/2; the table holds
// 2^(j / 64), and e^r with r = f ln2 / 64 (|r| <= 0.0055) is its Taylor
// polynomial of degree 5 (remainder below 1e-16).
__device__ __forceinline__ double exp2_64th(double y, const double* table) {
  if (y < -64.0 * 1000.0) return 0.0;
  const double shifted = y + 6755399441055744.0;  // 1.5 · 2^52: rounds to a whole number, held in the low bits
  const int k = __double2loint(shifted);
  const double r = (y - (shifted - 6755399441055744.0)) * (0.693147180559945309417 / 64.0);
  double e = __fma_rn(r, 1.0 / 120.0, 1.0 / 24.0);
  e = __fma_rn(e, r, 1.0 / 6.0);
  e = __fma_rn(e, r, 0.5);
  e = __fma_rn(e, r, 1.0);
  e = __fma_rn(e, r, 1.0);
  e *= table[k & 63];
  return __hiloint2double(__double2hiint(e) + ((k >> 6) << 20), __double2loint(e));  // e in [0.99, 2), k / 64 >= -1000
}

struct VerifyShared {
  float top[2][VERIFY_MAX_CLUSTER * VERIFY_WARPS];  // every warp's results of a round, in turn
  float sum[2][VERIFY_MAX_CLUSTER * VERIFY_WARPS];
  int at[2][VERIFY_MAX_CLUSTER * VERIFY_WARPS];  // greedy: the maximum's lowest id; else 0 when an id is allowed, INT_MAX when none
  double draw[2][VERIFY_MAX_CLUSTER * VERIFY_WARPS];
  float row_top[VERIFY_MAX_ROWS];
  int row_at[VERIFY_MAX_ROWS];
  bool row_accept[VERIFY_MAX_ROWS];
  double table[64];
};

template <typename T, bool GREEDY>
__global__ void __launch_bounds__(VERIFY_THREADS, 2) k_verify(VerifyDev v, int at_once) {
  constexpr int N = LogitRow<T>::N;
  __shared__ VerifyShared sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int s = blockIdx.x / ranks, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int words = (v.vocab + 31) / 32, pieces = LogitRow<T>::pieces(v.vocab), share = (pieces + ranks - 1) / ranks;
  const int lo = min(pieces, rank * share), hi = min(pieces, lo + share);
  const int drafts = v.draft_counts ? max(0, min(v.drafts, v.draft_counts[s])) : v.drafts;
  const double inverse = GREEDY ? 1.0 : 1.0 / (double)v.temperature;
  const float step = (float)(inverse * 1.4426950408889634);
  if (!GREEDY && tid < 64) sh.table[tid] = exp2((double)tid / 64.0);
  auto row_of = [&](int i, bool unmasked) {
    return LogitRow<T>(static_cast<const T*>(v.logits) + ((long long)s * (v.drafts + 1) + i) * v.row_stride,
                       v.mask && !unmasked ? v.mask + ((size_t)s * (v.drafts + 1) + i) * words : nullptr, v.vocab);
  };

  const int row_warps = VERIFY_WARPS / at_once;
  int turn = 0, kept = 0, best = 0;
  float top = -INFINITY;
  uint32_t unmasked = 0;  // rows of the round whose mask allows nothing
  bool stop = false;
  for (int i0 = 0; !stop;) {
    const int mine = warp / row_warps;
    {
      const int i = i0 + mine;
      float m = -INFINITY, sum = 0.0f;
      int where = INT_MAX;
      bool any = false;
      if (i <= drafts) {
        const LogitRow<T> row = row_of(i, unmasked >> mine & 1);
        constexpr int AHEAD = 4;
        const int stride = row_warps * 32;
        for (int c0 = lo + (warp % row_warps) * 32 + lane; c0 < hi; c0 += AHEAD * stride) {
          uint4 w[AHEAD];
#pragma unroll
          for (int a = 0; a < AHEAD; ++a)
            if (c0 + a * stride < hi) w[a] = row.raw(c0 + a * stride);
#pragma unroll
          for (int a = 0; a < AHEAD; ++a) {
            const int c = c0 + a * stride;
            if (c >= hi) break;
            float x[N];
            LogitRow<T>::widen_piece(w[a], x);
            const bool plain = !row.allowed && row.whole(c);
            const uint32_t bits = plain ? (1u << N) - 1 : row.live(c);
            any = any || bits;
            float high = -INFINITY;
#pragma unroll
            for (int e = 0; e < N; ++e) {
              x[e] = plain || (bits >> e & 1) ? tame(x[e]) : -INFINITY;
              high = fmaxf(high, x[e]);
            }
            if (high > m) {
              if (!GREEDY) sum = __fmul_rn(sum, exp2_fast(__fmul_rn(__fadd_rn(m, -high), step)));
              m = high;
              if (GREEDY) {
#pragma unroll
                for (int e = N - 1; e >= 0; --e)
                  if (x[e] == high) where = row.start(c) + e;
              }
            }
            if (!GREEDY && m != -INFINITY) {
              float add = 0.0f;
#pragma unroll
              for (int e = 0; e < N; ++e) add = __fadd_rn(add, exp2_fast(__fmul_rn(__fadd_rn(x[e], -m), step)));
              sum = __fadd_rn(sum, add);
            }
          }
        }
      }
      float wm = m;
#pragma unroll
      for (int o = 16; o; o >>= 1) wm = fmaxf(wm, __shfl_xor_sync(FULL, wm, o));
      int wat;
      if (GREEDY) {
        // a row of -inf alone has ids, but none to choose
        wat = __reduce_min_sync(FULL, m == wm ? (where == INT_MAX && any ? INT_MAX - 1 : where) : INT_MAX);
      } else {
        wat = __any_sync(FULL, any) ? 0 : INT_MAX;
        sum = m == -INFINITY ? 0.0f : __fmul_rn(sum, exp2_fast(__fmul_rn(__fadd_rn(m, -wm), step)));
#pragma unroll
        for (int o = 16; o; o >>= 1) sum = __fadd_rn(sum, __shfl_xor_sync(FULL, sum, o));
      }
      if (lane < ranks) {
        const int k = rank * VERIFY_WARPS + warp;
        *cluster.map_shared_rank(&sh.top[turn][k], lane) = wm;
        *cluster.map_shared_rank(&sh.at[turn][k], lane) = wat;
        if (!GREEDY) *cluster.map_shared_rank(&sh.sum[turn][k], lane) = sum;
      }
    }
    cluster.sync();
    // warp r joins the round's row r and decides on its draft
    if (warp < at_once && i0 + warp <= drafts) {
      const int i = i0 + warp, count = ranks * row_warps;
      auto entry = [&](int k) { return (k / row_warps) * VERIFY_WARPS + warp * row_warps + k % row_warps; };
      float m = -INFINITY;
      for (int k = lane; k < count; k += 32) m = fmaxf(m, sh.top[turn][entry(k)]);
#pragma unroll
      for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(FULL, m, o));
      int at = INT_MAX;
      double total = 0.0;
      for (int k = lane; k < count; k += 32) {
        const float t = sh.top[turn][entry(k)];
        if (!GREEDY || t == m) at = min(at, sh.at[turn][entry(k)]);
        if (!GREEDY && t != -INFINITY) total += (double)sh.sum[turn][entry(k)] * (double)exp2f(__fmul_rn(__fadd_rn(t, -m), step));
      }
      at = __reduce_min_sync(FULL, at);
      bool accept = false;
      if (i < drafts) {
        const uint32_t d = v.draft_tokens[(size_t)s * v.drafts + i];
        if (GREEDY) {
          accept = d == (uint32_t)at;
        } else {
#pragma unroll
          for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(FULL, total, o);
          const LogitRow<T> row = row_of(i, unmasked >> warp & 1);
          if (d < (uint32_t)v.vocab && m != -INFINITY && row.permits((int)d)) {
            const double p = exp(((double)tame(to_f32(row.p[d])) - (double)m) * inverse) / total;
            const double q = v.q ? (double)v.q[((size_t)s * v.drafts + i) * v.vocab + d] : 1.0;
            accept = (double)v.accept[(size_t)s * v.drafts + i] * q < p;
          }
        }
      }
      if (lane == 0) {
        sh.row_top[warp] = m;
        sh.row_at[warp] = at;
        sh.row_accept[warp] = accept;
      }
    }
    __syncthreads();
    uint32_t again = 0;
    for (int r = 0; r < at_once && !stop; ++r) {
      if (sh.row_at[r] == INT_MAX && !(unmasked >> r & 1)) {
        again = 1u << r;  // the mask allows nothing: all ids
        break;
      }
      top = sh.row_top[r];
      best = sh.row_at[r];
      stop = top == -INFINITY || !sh.row_accept[r];
      if (!stop) ++kept;
    }
    // the other set next: a slower CTA may still read this one
    turn ^= 1;
    if (again) {
      kept = i0;  // the round once more, with that row unmasked
      unmasked |= again;
    } else if (!stop) {
      i0 += at_once;
      unmasked = 0;
    } else {
      unmasked = unmasked >> (kept - i0) & 1;
    }
  }

  uint32_t* out = v.tokens + (size_t)s * (v.drafts + 1);
  if (rank == 0) {
    for (int i = tid; i <= v.drafts; i += VERIFY_THREADS) {
      if (i < kept) out[i] = v.draft_tokens[(size_t)s * v.drafts + i];
      if (i > kept || (i == kept && top == -INFINITY)) out[i] = NO_TOKEN;
      if (GREEDY && i == kept && top != -INFINITY) out[i] = (uint32_t)best;
    }
    if (tid == 0) v.accepted[s] = kept;
  }
  if (GREEDY || top == -INFINITY) {
    cluster.sync();  // no CTA leaves while another may write into its memory
    return;
  }

  // The draw. Warp w of a CTA takes the w-th run of the CTA's pieces; all
  // warps' sums go to every CTA, which finds the same warp; that warp finds
  // the id.
  const LogitRow<T> row = row_of(kept, unmasked);
  const int run = (hi - lo + VERIFY_WARPS - 1) / VERIFY_WARPS;
  const int from = min(hi, lo + warp * run), to = min(hi, from + run);
  const float* q = nullptr;
  int certain = -1;  // a draft without probabilities: q is 1 there
  if (kept < drafts) {
    if (v.q)
      q = v.q + ((size_t)s * v.drafts + kept) * v.vocab;
    else
      certain = (int)min(v.draft_tokens[(size_t)s * v.drafts + kept], (uint32_t)INT_MAX);
  }
  bool residual = kept < drafts;
  const double scale = inverse * (64.0 * 1.44269504088896340736);
  double over = 1.0;  // 1 / sum of the weights
  // a piece's weights, or with `less` what they have above q
  auto piece_shares = [&](int c, bool less, double (&x)[N]) {
    const uint4 w = row.raw(c);
    const uint32_t bits = row.live(c);
    const int e0 = row.start(c);
    float f[N];
    LogitRow<T>::widen_piece(w, f);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      double y = 0.0;
      if (bits >> e & 1) {
        const float t = tame(f[e]);
        if (t != -INFINITY) y = exp2_64th(((double)t - (double)top) * scale, sh.table);
        if (less) {
          const double minus = q ? (double)q[e0 + e] : e0 + e == certain ? 1.0 : 0.0;
          y = fmax(__fma_rn(y, over, -minus), 0.0);
        }
      }
      x[e] = y;
    }
  };
  auto all_sums = [&](bool less) {  // sh.draw[turn] = every warp's sum
    double mine = 0.0;
    for (int c = from + lane; c < to; c += 32) {
      double x[N];
      piece_shares(c, less, x);
#pragma unroll
      for (int e = 0; e < N; ++e) mine += x[e];
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(FULL, mine, o);
    if (lane < ranks) *cluster.map_shared_rank(&sh.draw[turn][rank * VERIFY_WARPS + warp], lane) = mine;
    cluster.sync();
  };
  const int count = ranks * VERIFY_WARPS;
  auto sum_up = [&] {
    double x = 0.0;
    for (int k = lane; k < count; k += 32) x += sh.draw[turn][k];
#pragma unroll
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(FULL, x, o);
    return x;
  };
  all_sums(false);
  double whole = sum_up();
  if (residual) {
    over = 1.0 / whole;
    const int first = turn;
    turn ^= 1;
    all_sums(true);
    const double left = sum_up();
    if (left > 0.0) {
      whole = left;
    } else {
      residual = false;  // p nowhere exceeds q: from p
      turn = first;
    }
  }
  const double goal = (double)v.sample[s] * whole;
  // the first warp whose running sum passes the goal; 4 neighbouring sums a lane
  double own[4], upto = 0.0;
  int last = -1;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    own[k] = lane * 4 + k < count ? sh.draw[turn][lane * 4 + k] : 0.0;
    if (own[k] > 0.0) last = lane * 4 + k;
    upto += own[k];
  }
  double before = upto;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double y = __shfl_up_sync(FULL, before, o);
    if (lane >= o) before += y;
  }
  before -= upto;
  int owner = INT_MAX;
  double ahead = before, at_owner = 0.0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (owner == INT_MAX && own[k] > 0.0 && ahead + own[k] > goal) {
      owner = lane * 4 + k;
      at_owner = ahead;
    }
    ahead += own[k];
  }
  const int chosen = __reduce_min_sync(FULL, owner);
  const bool end = chosen == INT_MAX;  // a uniform at the very end, or out of range: the last id with a share
  const int winner = end ? __reduce_max_sync(FULL, last) : chosen;
  before = __shfl_sync(FULL, at_owner, (winner >> 2) & 31);
  if (winner == rank * VERIFY_WARPS + warp) {
    int found = -1, final = -1;
    for (int c0 = from; c0 < to && found < 0; c0 += 32) {
      const int c = c0 + lane;
      double x[N], mine = 0.0;
      if (c < to) {
        piece_shares(c, residual, x);
#pragma unroll
        for (int e = 0; e < N; ++e) mine += x[e];
      }
      double up = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(FULL, up, o);
        if (lane >= o) up += y;
      }
      const double all = __shfl_sync(FULL, up, 31);
      double reach = before + (up - mine);
      int hit = INT_MAX, high = -1;
      if (c < to) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          reach += x[e];
          if (x[e] > 0.0) {
            high = row.start(c) + e;
            if (hit == INT_MAX && reach > goal) hit = high;
          }
        }
      }
      const int lowest = __reduce_min_sync(FULL, hit), highest = __reduce_max_sync(FULL, high);
      if (highest >= 0) final = highest;
      if (lowest != INT_MAX && !end) found = lowest;
      before += all;
    }
    // the order of summing may leave the border a rounding beyond the run's last id
    if (lane == 0) out[kept] = (uint32_t)(found >= 0 ? found : final);
  }
  cluster.sync();
}

cudaError_t verify_drafts(const VerifyDev& v, cudaStream_t st) {
  if (v.sequences == 0) return cudaSuccess;
  const int size = v.dtype == DTYPE_F32 ? 4 : 2;
  // CTAs for a sequence: until the 148 SMs hold two each, or a slice is 8 KB
  int ranks = 1;
  while (ranks < VERIFY_MAX_CLUSTER && v.sequences * ranks * 2 <= 2 * 148 && v.vocab * size / ranks > 8192) ranks *= 2;
  // rows of a round: until a CTA has 32 KB in flight
  int at_once = 1;
  while (at_once < VERIFY_MAX_ROWS && at_once < v.drafts + 1 && (long long)v.vocab * size / ranks * at_once * 2 <= 32768) at_once *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(v.sequences * ranks));
  cfg.blockDim = dim3(VERIFY_THREADS);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const bool greedy = v.temperature == 0.0f;
  if (v.dtype == DTYPE_F32) return cudaLaunchKernelEx(&cfg, greedy ? k_verify<float, true> : k_verify<float, false>, v, at_once);
  if (v.dtype == DTYPE_F16) return cudaLaunchKernelEx(&cfg, greedy ? k_verify<__half, true> : k_verify<__half, false>, v, at_once);
  return cudaLaunchKernelEx(&cfg, greedy ? k_verify<__nv_bfloat16, true> : k_verify<__nv_bfloat16, false>, v, at_once);
}

}  // namespace nbk
