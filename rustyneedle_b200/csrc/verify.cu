// verify.cu — drafted tokens against the target's probabilities.
//
// Row i of a sequence has p_i = softmax(x_i / T) over its allowed ids. Draft d
// is accepted while u_i · q_i(d) < p_i(d); at the first rejection the token is
// the lowest id whose running sum of max(p - q, 0) passes u · total, behind the
// last draft the same with p alone. The rows up to the first rejection are
// needed, those behind it are not read.
//
// One cluster of CTAs takes a sequence: each CTA a contiguous slice of the
// vocabulary, the rows one after another. A row's pass keeps a running maximum
// and sum for every thread (f32 exponentials, sums joined in f64), which decides
// the draft; the one row that a token is drawn from is read once or twice
// more, from L2, with exponentials and running sums in f64: a f32 sum of a
// large vocabulary would put some draws on the wrong side of a border.
#include <cooperative_groups.h>

#include <cfloat>

#include "serving.cuh"

namespace nbk {

namespace cg = cooperative_groups;

constexpr int VERIFY_THREADS = 512, VERIFY_WARPS = VERIFY_THREADS / 32, VERIFY_MAX_CLUSTER = 8;
constexpr uint32_t NO_TOKEN = 0xffffffffu;

// A logit as the formulas take it: NaN counts as -inf, +inf as the largest f32.
__device__ __forceinline__ float tame(float x) { return x != x ? -INFINITY : fminf(x, FLT_MAX); }

template <typename T>
__global__ void __launch_bounds__(VERIFY_THREADS) k_verify(VerifyDev v, int slice) {
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int s = blockIdx.x / ranks, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int lo = min(v.vocab, rank * slice), hi = min(v.vocab, lo + slice);
  const int words = (v.vocab + 31) / 32;
  const int drafts = v.draft_counts ? max(0, min(v.drafts, v.draft_counts[s])) : v.drafts;
  const bool greedy = v.temperature == 0.0f;
  const double inverse = greedy ? 1.0 : 1.0 / (double)v.temperature;
  const float step = (float)(inverse * 1.4426950408889634);

  __shared__ float w_top[VERIFY_WARPS];
  __shared__ int w_at[VERIFY_WARPS];
  __shared__ double w_sum[VERIFY_WARPS];
  __shared__ float r_top[2][VERIFY_MAX_CLUSTER];  // one set a row, every CTA's results, in turn
  __shared__ int r_at[2][VERIFY_MAX_CLUSTER];
  __shared__ double r_sum[2][VERIFY_MAX_CLUSTER];
  __shared__ double d_sum[2][VERIFY_MAX_CLUSTER * VERIFY_WARPS];  // the draw: every warp's sum, in turn

  int turn = 0, kept = 0;
  float top = -INFINITY;
  const T* row = nullptr;
  const uint32_t* allowed = nullptr;
  for (int i = 0;; ++i) {
    row = static_cast<const T*>(v.logits) + ((long long)s * (v.drafts + 1) + i) * v.row_stride;
    allowed = v.mask ? v.mask + ((size_t)s * (v.drafts + 1) + i) * words : nullptr;
    const bool last = i == drafts;
    const uint32_t d = last ? NO_TOKEN : v.draft_tokens[(size_t)s * v.drafts + i];
    double total = 0.0;
    int at = 0;
    for (;;) {
      // this thread's maximum (lowest id on ties) and sum
      float m = -INFINITY, sum = 0.0f;
      int where = INT_MAX;
      bool any = false;
      for (int t = lo + tid; t < hi; t += VERIFY_THREADS) {
        if (allowed && !(allowed[t >> 5] >> (t & 31) & 1)) continue;
        any = true;
        const float x = tame(to_f32(row[t]));
        if (x > m) {
          sum = __fmul_rn(sum, exp2f(__fmul_rn(__fadd_rn(m, -x), step)));
          m = x;
          where = t;
        }
        if (x != -INFINITY) sum = __fadd_rn(sum, exp2f(__fmul_rn(__fadd_rn(x, -m), step)));
      }
      // -inf with an id: something is allowed, but nothing has a probability
      if (any && where == INT_MAX) where = INT_MAX - 1;
      float wm = m;
      for (int o = 16; o; o >>= 1) wm = fmaxf(wm, __shfl_xor_sync(FULL, wm, o));
      int wat = m == wm ? where : INT_MAX;
      wat = __reduce_min_sync(FULL, wat);
      double ws = m == -INFINITY ? 0.0 : (double)sum * exp2((double)(m - wm) * (double)step);
      for (int o = 16; o; o >>= 1) ws += __shfl_xor_sync(FULL, ws, o);
      if (lane == 0) {
        w_top[warp] = wm;
        w_at[warp] = wat;
        w_sum[warp] = ws;
      }
      __syncthreads();
      if (tid == 0) {
        float cm = -INFINITY;
        for (int w = 0; w < VERIFY_WARPS; ++w) cm = fmaxf(cm, w_top[w]);
        int cat = INT_MAX;
        double cs = 0.0;
        for (int w = 0; w < VERIFY_WARPS; ++w) {
          if (w_top[w] == cm) cat = min(cat, w_at[w]);
          if (w_top[w] != -INFINITY) cs += w_sum[w] * exp2((double)(w_top[w] - cm) * (double)step);
        }
        for (int r = 0; r < ranks; ++r) {
          *cluster.map_shared_rank(&r_top[turn][rank], r) = cm;
          *cluster.map_shared_rank(&r_at[turn][rank], r) = cat;
          *cluster.map_shared_rank(&r_sum[turn][rank], r) = cs;
        }
      }
      cluster.sync();
      top = -INFINITY;
      for (int r = 0; r < ranks; ++r) top = fmaxf(top, r_top[turn][r]);
      at = INT_MAX;
      total = 0.0;
      for (int r = 0; r < ranks; ++r) {
        if (r_top[turn][r] == top) at = min(at, r_at[turn][r]);
        if (r_top[turn][r] != -INFINITY) total += r_sum[turn][r] * exp2((double)(r_top[turn][r] - top) * (double)step);
      }
      turn ^= 1;  // the other set: a slower CTA may still read this one
      if (at != INT_MAX || !allowed) break;
      allowed = nullptr;  // the mask allows nothing: all ids
    }
    if (top == -INFINITY) break;  // nothing left to accept or to draw
    bool accept = false;
    if (!last && d < (uint32_t)v.vocab) {
      if (greedy) {
        accept = (int)d == at;
      } else if (!allowed || (allowed[d >> 5] >> (d & 31) & 1)) {
        const double p = exp(((double)tame(to_f32(row[d])) - (double)top) * inverse) / total;
        const double q = v.q ? (double)v.q[((size_t)s * v.drafts + i) * v.vocab + d] : 1.0;
        accept = (double)v.accept[(size_t)s * v.drafts + i] * q < p;
      }
    }
    if (!accept) {
      if (greedy && rank == 0 && tid == 0) v.tokens[(size_t)s * (v.drafts + 1) + i] = (uint32_t)at;
      break;
    }
    ++kept;
  }
  uint32_t* out = v.tokens + (size_t)s * (v.drafts + 1);
  if (rank == 0) {
    for (int i = tid; i <= v.drafts; i += VERIFY_THREADS) {
      if (i < kept) out[i] = v.draft_tokens[(size_t)s * v.drafts + i];
      if (i > kept || (i == kept && top == -INFINITY)) out[i] = NO_TOKEN;
    }
    if (tid == 0) v.accepted[s] = kept;
  }
  if (greedy || top == -INFINITY) {
    cluster.sync();  // no CTA leaves while another may write into its memory
    return;
  }

  // The draw. Warp w of CTA r takes the w-th run of the CTA's slice; all warps'
  // sums go to every CTA, which finds the same warp; that warp finds the id.
  const int run = ((hi - lo + VERIFY_WARPS - 1) / VERIFY_WARPS + 31) / 32 * 32;
  const int from = min(hi, lo + warp * run), to = min(hi, from + run);
  const float* q = nullptr;
  uint32_t certain = NO_TOKEN;  // a draft without probabilities: q is 1 there
  if (kept < drafts) {
    if (v.q)
      q = v.q + ((size_t)s * v.drafts + kept) * v.vocab;
    else
      certain = v.draft_tokens[(size_t)s * v.drafts + kept];
  }
  auto weight = [&](int t) -> double {
    if (allowed && !(allowed[t >> 5] >> (t & 31) & 1)) return 0.0;
    return exp(((double)tame(to_f32(row[t])) - (double)top) * inverse);
  };
  auto all_sums = [&](double mine) {  // d_sum[turn] = every warp's sum over its lanes
    for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(FULL, mine, o);
    if (lane < ranks) *cluster.map_shared_rank(&d_sum[turn][rank * VERIFY_WARPS + warp], lane) = mine;
    cluster.sync();
  };
  auto sum_up = [&] {
    double x = 0.0;
    for (int k = 0; k < ranks * VERIFY_WARPS; ++k) x += d_sum[turn][k];
    return x;
  };
  double total = 1.0, sum = 0.0;
  if (q || certain != NO_TOKEN) {
    for (int t = from + lane; t < to; t += 32) sum += weight(t);
    all_sums(sum);
    total = sum_up();
    turn ^= 1;
    sum = 0.0;
  }
  bool residual = q || certain != NO_TOKEN;
  auto share = [&](int t) -> double {
    const double p = weight(t);
    if (!residual) return p;
    const double less = q ? (double)q[t] : (uint32_t)t == certain ? 1.0 : 0.0;
    const double x = p / total - less;
    return x > 0.0 ? x : 0.0;
  };
  double whole;
  for (;;) {
    for (int t = from + lane; t < to; t += 32) sum += share(t);
    all_sums(sum);
    whole = sum_up();
    if (whole > 0.0 || !residual) break;
    turn ^= 1;
    residual = false;  // p nowhere exceeds q
    sum = 0.0;
  }
  const double goal = (double)v.sample[s] * whole;
  int owner = -1, last = 0;
  double before = 0.0, upto = 0.0;
  for (int k = 0; k < ranks * VERIFY_WARPS; ++k) {
    const double x = d_sum[turn][k];
    if (x > 0.0) last = k;
    if (owner < 0) {
      before = upto;
      upto += x;
      if (upto > goal) owner = k;
    }
  }
  const bool end = owner < 0;  // a uniform at the very end, or out of range: the last id with a share
  if (end) owner = last;
  if (owner == rank * VERIFY_WARPS + warp) {
    int found = -1, final = -1;
    for (int t0 = from; t0 < to && found < 0; t0 += 32) {
      const int t = t0 + lane;
      const double x = t < to ? share(t) : 0.0;
      double up = x;
      for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(FULL, up, o);
        if (lane >= o) up += y;
      }
      const unsigned some = __ballot_sync(FULL, x > 0.0);
      if (some) final = t0 + 31 - __clz(some);
      const unsigned past = __ballot_sync(FULL, x > 0.0 && before + up > goal);
      if (past && !end) found = t0 + __ffs(past) - 1;
      before += __shfl_sync(FULL, up, 31);
    }
    // the lanes' order of summing may leave the border a rounding beyond the run's last id
    if (lane == 0) out[kept] = (uint32_t)(found >= 0 ? found : final);
  }
  cluster.sync();
}

cudaError_t verify_drafts(const VerifyDev& v, cudaStream_t st) {
  if (v.sequences == 0) return cudaSuccess;
  int ranks = 1;
  while (ranks < VERIFY_MAX_CLUSTER && v.sequences * ranks < 296 && v.vocab / ranks > 4096) ranks *= 2;
  const int slice = ((v.vocab + ranks - 1) / ranks + 31) / 32 * 32;
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
  if (v.dtype == DTYPE_F32) return cudaLaunchKernelEx(&cfg, k_verify<float>, v, slice);
  if (v.dtype == DTYPE_F16) return cudaLaunchKernelEx(&cfg, k_verify<__half>, v, slice);
  return cudaLaunchKernelEx(&cfg, k_verify<__nv_bfloat16>, v, slice);
}

}  // namespace nbk
