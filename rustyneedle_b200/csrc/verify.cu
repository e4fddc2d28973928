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
// border. So they would some acceptances: where u · q and p are closer than the
// f32 sum's error (about one draft in 10000), the round is gone through again
// with that row's sum in f64.
#include <cooperative_groups.h>

#include <cfloat>
#include <type_traits>

#include "serving.cuh"

namespace nbk {

namespace cg = cooperative_groups;

constexpr int VERIFY_MAX_CLUSTER = 8, VERIFY_MAX_ROWS = 8, VERIFY_MAX_WARPS = 16;
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
  __host__ __device__ static int pieces(int v) { return v / N + 2; }
  __device__ __forceinline__ int start(int piece) const { return head + (piece - 1) * N; }
  // pieces [1, whole_end()) lie whole within the row
  __device__ __forceinline__ int whole_end() const { return (vocab - head) / N + 1; }
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
    const uint32_t word[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (N == 4) {
        x[i] = __uint_as_float(word[i]);
      } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        x[2 * i] = __uint_as_float(word[i] << 16);
        x[2 * i + 1] = __uint_as_float(word[i] & 0xffff0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&word[i]));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      }
    }
  }
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 2^(y / 128) for -128000 <= y <= 0 in f64, a table-driven exponential after
// P. T. P. Tang (1989): y = k + f, k whole, |f| <= 1/2; the table holds 2^(j / 128), sixteen times over so that no two lanes of a half
// warp meet in a bank, and 2^(f / 128) = e^r with r = f ln2 / 128 (|r| <=
// 0.0028) is its Taylor polynomial of degree 3, within 3e-12 relative. The
// power of two goes into the table's value: 2^(y / 128) = e · t. Entry j's high
// word is kept less j 2^13, so that adding k 2^13 leaves k / 128 in the exponent.
constexpr int EXP_ENTRIES = 128, EXP_COPIES = 16;
struct Exp2Table {
  double entry[EXP_ENTRIES];
};
// 2^(j / 128) by the exponential's series, and its high word less j 2^13. The
// high word is at least 0x3ff00000 - 127 · 2^13 > 0 and the sum below restores
// it, so the entry is taken apart only as bits.
constexpr Exp2Table exp2_table() {
  Exp2Table t{};
  for (int j = 0; j < EXP_ENTRIES; ++j) {
    const double r = j * (0.693147180559945309417 / EXP_ENTRIES);
    double sum = 1.0;
    for (int n = 24; n > 0; --n) sum = 1.0 + sum * r / n;
    // sum = 1 + m 2^-52 with a whole m; taking j 2^13 from the high word takes
    // j 2^-7 from the mantissa, and one from the exponent where that borrows
    const double less = j / 128.0, mantissa = sum - 1.0;
    t.entry[j] = mantissa >= less ? 1.0 + (mantissa - less) : 0.5 * (1.0 + (mantissa - less + 1.0));
  }
  return t;
}
__device__ const Exp2Table g_exp2_table = exp2_table();

struct Exp2Parts {
  double e, t;
};
__device__ __forceinline__ Exp2Parts exp2_128th(double y, const double* table) {
  constexpr double C = 0.693147180559945309417 / EXP_ENTRIES, C2 = C * C / 2.0, C3 = C2 * C / 3.0;
  const double shifted = y + 6755399441055744.0;  // 1.5 · 2^52: rounds to a whole number, held in the low bits
  const int k = __double2loint(shifted);
  const double f = y - (shifted - 6755399441055744.0);
  Exp2Parts x;
  x.e = __fma_rn(f, C3, C2);
  x.e = __fma_rn(x.e, f, C);
  x.e = __fma_rn(x.e, f, 1.0);
  const double t = *reinterpret_cast<const double*>(reinterpret_cast<const char*>(table) + ((k << 7) & ((EXP_ENTRIES - 1) << 7)));
  x.t = __hiloint2double(__double2hiint(t) + (k << (20 - 7)), __double2loint(t));  // k / 128 >= -1000
  return x;
}

// A thread's part of a row: the maximum (greedy: and its lowest id) and the sum
// of e^((x - m) / T). `base` is fl(m step) and `shift` 2^(base - m step): a
// weight is 2^(x step - base), one multiply-add and one exponential, and the
// sum of a batch comes to m by one product.
template <bool GREEDY>
struct RowStats {
  float m = -INFINITY, sum = 0.0f, base = 0.0f, shift = 1.0f;
  int where = INT_MAX;
  bool any = false;  // an id is allowed
};
constexpr float BASE_MOST = 32768.0f;  // beyond it, base is too coarse for the product

// Twice the largest relative error of a row's sum, in units of 2^-24, where a
// thread adds up `batches` batches of at most 64 weights. A weight 2^-a comes
// from three roundings of a (the step, the product, the difference) and ex2,
// within 2^-22; the mean of a over the weights is at most log2 vocab <= 24, so
// that is 24 · 3 · ln 2 + 4 = 54, and as much again where a thread's sum comes
// to its warp's maximum and a warp's to the row's. Adding up: 64 for a batch, 8
// for the shift and the warp, and for every batch 8 for the sum's own rescaling
// and addition. In all 3 · 54 + 72 < 256, and 8 a batch.
static double sum_slack(int batches) { return (512 + 16 * batches) * 0x1p-24; }
enum Verdict : int { REJECTED, ACCEPTED, UNSURE };

// The pieces c, c + stride, .. below `end`, A of them at once so that their
// loads overlap and the maximum is looked at once for all. CLEAN: they are
// whole and no id is masked.
template <typename T, bool GREEDY, int A, bool CLEAN>
__device__ __forceinline__ void take_pieces(const LogitRow<T>& row, int c, int stride, int end, float step, RowStats<GREEDY>& st) {
  constexpr int N = LogitRow<T>::N;
  constexpr uint32_t NONE = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;  // -inf
  uint4 w[A];
  uint32_t bits[A];
#pragma unroll
  for (int a = 0; a < A; ++a) {
    const int k = c + a * stride;
    w[a] = make_uint4(NONE, NONE, NONE, NONE);
    bits[a] = 0;
    if (CLEAN) {
      if (k < end) w[a] = *reinterpret_cast<const uint4*>(row.p + row.start(k));
    } else {
      if (k < end) w[a] = row.raw(k), bits[a] = row.live(k);
    }
  }
  if constexpr (GREEDY && CLEAN && N == 8) {
    // Nearly every step has nothing above the maximum: two values an
    // instruction, NaN dropped, and room for eight loads in flight (200 rows of
    // 50257: 37.6 us, with four 41.4).
    using Pair = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    Pair pair;
    memcpy(&pair, &w[0].x, 4);
#pragma unroll
    for (int a = 0; a < A; ++a) {
      Pair at[4];
      memcpy(at, &w[a], 16);
#pragma unroll
      for (int i = 0; i < 4; ++i) pair = __hmax2(pair, at[i]);
    }
    st.any = true;
    const float high = fmaxf(to_f32(pair.x), to_f32(pair.y));
    // 64 NaNs leave a NaN, which is no maximum: it must not reach fminf, which
    // would drop it for FLT_MAX
    if (!(high > st.m) || st.m == FLT_MAX) return;
    st.m = fminf(high, FLT_MAX);  // no 16-bit value but +inf comes to FLT_MAX
#pragma unroll
    for (int a = A - 1; a >= 0; --a) {
      float t[N];
      LogitRow<T>::widen_piece(w[a], t);
#pragma unroll
      for (int e = N - 1; e >= 0; --e)
        if (t[e] == high) st.where = row.start(c + a * stride) + e;
    }
    return;
  }
  float x[A * N];
#pragma unroll
  for (int a = 0; a < A; ++a) {
    float t[N];
    LogitRow<T>::widen_piece(w[a], t);
#pragma unroll
    for (int e = 0; e < N; ++e) x[a * N + e] = CLEAN ? t[e] : bits[a] >> e & 1 ? tame(t[e]) : -INFINITY;
    st.any = st.any || CLEAN || bits[a];
  }
  float high = x[0];
#pragma unroll
  for (int e = 1; e < A * N; ++e) high = fmaxf(high, x[e]);  // drops NaN
  if (high > st.m) {
    if (CLEAN && high > FLT_MAX) {  // +inf among them
#pragma unroll
      for (int e = 0; e < A * N; ++e) x[e] = tame(x[e]);
      high = FLT_MAX;
    }
    if (!GREEDY) {
      st.sum = __fmul_rn(st.sum, exp2_fast(__fmul_rn(__fadd_rn(st.m, -high), step)));
      st.base = __fmul_rn(high, step);
      st.shift = exp2_fast(-__fmaf_rn(high, step, -st.base));
    } else if (high > st.m) {
#pragma unroll
      for (int e = A * N - 1; e >= 0; --e)
        if (x[e] == high) st.where = row.start(c + e / N * stride) + e % N;
    }
    st.m = high;
  }
  if (!GREEDY && st.m != -INFINITY) {
    float add = 0.0f;
    const float base = st.base;
    if (fabsf(base) <= BASE_MOST) {
#pragma unroll
      for (int e = 0; e < A * N; ++e) add = __fadd_rn(add, exp2_fast(__fmaf_rn(x[e], step, -base)));
      add = __fmul_rn(add, st.shift);
    }
    if (!(fabsf(base) <= BASE_MOST) || add != add) {  // very large logits, or a NaN among them
      add = 0.0f;
#pragma unroll
      for (int e = 0; e < A * N; ++e) add = __fadd_rn(add, exp2_fast(__fmul_rn(__fadd_rn(tame(x[e]), -st.m), step)));
    }
    st.sum = __fadd_rn(st.sum, add);
  }
}

constexpr int DRAFTS = 64;  // whose numbers are held at once, a multiple of the rows of a round
constexpr int DRAW_GROUPS = 4;
constexpr double FLOOR = -124000.0;                    // of exp2_128th's argument: 2^-968
constexpr double GHOST = 1e-289, GHOSTS = 1e-280;  // a share, a sum of shares, that counts as none

// A piece as it lies in memory, its live ids, and the draft's probabilities.
template <int N>
struct Piece {
  uint4 w;
  uint32_t bits;
  float q[N];
};
struct Draw {
  const double* table;
  float lowest, top;
  double scale;  // (x - top) · scale is the exponential's argument
  double lift;   // 128 log2 of 1 / the sum of the weights, once that is known
  double offset; // lift - top · scale, where that is small enough to be exact
};

// A piece's weights, or (LESS) what the probabilities have above q; without
// branches, so that the chains of several elements overlap. ALL: every id is
// live, and the logits are of a size (2^30 of the exponential's steps) whose
// product with the scale is off by 2^-23 of a step at most, the same for all.
template <typename T, bool LESS, bool ALL>
__device__ __forceinline__ void piece_shares(const Piece<LogitRow<T>::N>& p, const Draw& d, double (&x)[LogitRow<T>::N]) {
  constexpr int N = LogitRow<T>::N;
  float f[N];
  LogitRow<T>::widen_piece(p.w, f);
  const double top = d.top;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    float t = fmaxf(f[e], d.lowest);
    if (!ALL) t = fminf(t, d.top);
    double y = ALL ? __fma_rn((double)t, d.scale, d.offset) : __fma_rn((double)t - top, d.scale, d.lift);
    if (!ALL) y = (p.bits >> e & 1) && f[e] > -INFINITY ? y : FLOOR;
    const Exp2Parts w = exp2_128th(y, d.table);
    if (LESS) {
      const double r = __fma_rn(w.e, w.t, -(double)p.q[e]);
      x[e] = __double2hiint(r) < 0 ? 0.0 : r;  // a NaN stays
    } else {
      x[e] = w.e * w.t;
    }
  }
}

struct VerifyShared {
  float top[2][VERIFY_MAX_CLUSTER * VERIFY_MAX_WARPS];  // every warp's results of a round, in turn
  float sum[2][VERIFY_MAX_CLUSTER * VERIFY_MAX_WARPS];
  int at[2][VERIFY_MAX_CLUSTER * VERIFY_MAX_WARPS];  // greedy: the maximum's lowest id; else 0 when an id is allowed, INT_MAX when none
  double draw[2][VERIFY_MAX_CLUSTER * VERIFY_MAX_WARPS];
  double group[2][VERIFY_MAX_WARPS][DRAW_GROUPS];  // this CTA's: sums of a warp's run, piece by piece
  float row_top[VERIFY_MAX_ROWS];
  int row_at[VERIFY_MAX_ROWS];
  uint32_t draft[DRAFTS];
  float draft_logit[DRAFTS], draft_q[DRAFTS], uniform[DRAFTS];
  int draft_allowed[DRAFTS];
  Verdict row_verdict[VERIFY_MAX_ROWS];
  double table[EXP_ENTRIES * EXP_COPIES];
};

__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
  for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(FULL, x, o);
  return x;
}

// slack: sum_slack of the launch's rows
template <typename T, bool GREEDY, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, 32 / WARPS) k_verify(VerifyDev v, int at_once, double slack) {
  constexpr int N = LogitRow<T>::N;
  __shared__ VerifyShared sh;
  cg::cluster_group cluster = cg::this_cluster();
  cluster_arrive_relaxed();  // paired with the wait before the first remote store
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int s = blockIdx.x / ranks, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int words = (v.vocab + 31) / 32, pieces = LogitRow<T>::pieces(v.vocab), share = (pieces + ranks - 1) / ranks;
  const int lo = min(pieces, rank * share), hi = min(pieces, lo + share);
  const int drafts = v.draft_counts ? max(0, min(v.drafts, v.draft_counts[s])) : v.drafts;
  const double inverse = GREEDY ? 1.0 : 1.0 / (double)v.temperature;
  const float step = (float)(inverse * 1.4426950408889634);
  if (!GREEDY)
    for (int i = tid; i < EXP_ENTRIES * EXP_COPIES; i += (WARPS * 32)) sh.table[i] = g_exp2_table.entry[i / EXP_COPIES];
  auto row_of = [&](int i, bool unmasked) {
    return LogitRow<T>(static_cast<const T*>(v.logits) + ((long long)s * (v.drafts + 1) + i) * v.row_stride,
                       v.mask && !unmasked ? v.mask + ((size_t)s * (v.drafts + 1) + i) * words : nullptr, v.vocab);
  };

  const int row_warps = WARPS / at_once;
  int turn = 0, kept = 0, best = 0;
  float top = -INFINITY;
  uint32_t unmasked = 0;  // rows of the round whose mask allows nothing
  uint32_t exact = 0;     // rows of the round whose sums are formed in f64
  bool stop = false, redo = false, alone = true;  // alone: the cluster's other CTAs may not run yet
  for (int i0 = 0; !stop;) {
    const int mine = warp / row_warps;
    // what the decisions need of the drafts, DRAFTS rows ahead: two dependent
    // loads from far, taken once by the last warps
    if (i0 % DRAFTS == 0 && !redo && tid >= WARPS * 32 - DRAFTS) {
      const int k = tid - (WARPS * 32 - DRAFTS), i = i0 + k;
      if (i < drafts) {
        const size_t at = (size_t)s * v.drafts + i;
        const uint32_t d = v.draft_tokens[at];
        sh.draft[k] = d;
        if (!GREEDY) {
          sh.uniform[k] = v.accept[at];
          const bool known = d < (uint32_t)v.vocab;
          const LogitRow<T> row = row_of(i, true);
          sh.draft_logit[k] = known ? tame(to_f32(row.p[d])) : -INFINITY;
          sh.draft_q[k] = known && v.q ? v.q[at * v.vocab + d] : 1.0f;
          sh.draft_allowed[k] = known && v.mask ? v.mask[((size_t)s * (v.drafts + 1) + i) * words + (d >> 5)] >> (d & 31) & 1 : 1;
        }
      }
    }
    {
      const int i = i0 + mine;
      RowStats<GREEDY> st;
      if (!GREEDY && exact >> mine & 1) {
        st.m = sh.row_top[mine];  // of the pass before
        st.any = true;
      } else if (i <= drafts) {
        const LogitRow<T> row = row_of(i, unmasked >> mine & 1);
        const int stride = row_warps * 32;
        int c = lo + (warp % row_warps) * 32 + lane;
        if (!row.allowed) {
          if (c == 0) take_pieces<T, GREEDY, 1, false>(row, 0, stride, hi, step, st), c += stride;
          constexpr int A = N == 8 && !GREEDY ? 4 : 8;
          const int whole = min(hi, row.whole_end());
          for (; c < whole; c += A * stride) take_pieces<T, GREEDY, A, true>(row, c, stride, whole, step, st);
          // what is left are the row's last pieces, short or empty
          if (whole < hi && tid % (row_warps * 32) == 0)
            for (int k = max(lo, whole); k < hi; ++k) take_pieces<T, GREEDY, 1, false>(row, k, 1, hi, step, st);
        } else {
          for (; c < hi; c += 4 * stride) take_pieces<T, GREEDY, 4, false>(row, c, stride, hi, step, st);
        }
      }
      const float m = st.m;
      float sum = st.sum;
      float wm = m;
#pragma unroll
      for (int o = 16; o; o >>= 1) wm = fmaxf(wm, __shfl_xor_sync(FULL, wm, o));
      int wat;
      if (GREEDY) {
        // a row of -inf alone has ids, but none to choose
        wat = __reduce_min_sync(FULL, m == wm ? (st.where == INT_MAX && st.any ? INT_MAX - 1 : st.where) : INT_MAX);
      } else {
        wat = __any_sync(FULL, st.any) ? 0 : INT_MAX;
        sum = m == -INFINITY ? 0.0f : __fmul_rn(sum, exp2_fast(__fmul_rn(__fadd_rn(m, -wm), step)));
#pragma unroll
        for (int o = 16; o; o >>= 1) sum = __fadd_rn(sum, __shfl_xor_sync(FULL, sum, o));
      }
      if (alone) {
        __syncwarp();
        cluster_wait();  // every CTA of the cluster runs: its shared memory is usable
        alone = false;
      }
      if (!GREEDY && __builtin_expect(exact >> mine & 1, 0)) {
        const LogitRow<T> row = row_of(i, unmasked >> mine & 1);
        const int threads = row_warps * 32;
        double precise = 0.0;
#pragma unroll 1
        for (int id = rank * threads + tid % threads; id < v.vocab; id += ranks * threads)
          if (row.permits(id)) precise += exp(((double)tame(to_f32(row.p[id])) - (double)m) * inverse);
        precise = warp_sum(precise);
        if (lane < ranks) *cluster.map_shared_rank(&sh.draw[turn][rank * WARPS + warp], lane) = precise;
      }
      if (lane < ranks) {
        const int k = rank * WARPS + warp;
        *cluster.map_shared_rank(&sh.top[turn][k], lane) = wm;
        *cluster.map_shared_rank(&sh.at[turn][k], lane) = wat;
        if (!GREEDY) *cluster.map_shared_rank(&sh.sum[turn][k], lane) = sum;
      }
    }
    cluster.sync();
    // warp r joins the round's row r and decides on its draft
    if (warp < at_once && i0 + warp <= drafts) {
      const int i = i0 + warp, count = ranks * row_warps;
      auto entry = [&](int k) { return (k / row_warps) * WARPS + warp * row_warps + k % row_warps; };
      float m = -INFINITY;
      for (int k = lane; k < count; k += 32) m = fmaxf(m, sh.top[turn][entry(k)]);
#pragma unroll
      for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(FULL, m, o));
      int at = INT_MAX;
      double total = 0.0;
      for (int k = lane; k < count; k += 32) {
        const float t = sh.top[turn][entry(k)];
        if (!GREEDY || t == m) at = min(at, sh.at[turn][entry(k)]);
        if (!GREEDY && exact >> warp & 1)
          total += sh.draw[turn][entry(k)];
        else if (!GREEDY && t != -INFINITY)
          total += (double)sh.sum[turn][entry(k)] * (double)exp2f(__fmul_rn(__fadd_rn(t, -m), step));
      }
      at = __reduce_min_sync(FULL, at);
      Verdict verdict = REJECTED;
      if (i < drafts) {
        if (GREEDY) {
          verdict = sh.draft[i % DRAFTS] == (uint32_t)at ? ACCEPTED : REJECTED;
        } else {
#pragma unroll
          for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(FULL, total, o);
          const int k = i % DRAFTS;
          const float x = sh.draft_logit[k];
          if (x != -INFINITY && (sh.draft_allowed[k] || (unmasked >> warp & 1))) {
            const double left = (double)sh.uniform[k] * (double)sh.draft_q[k] * total, right = exp(((double)x - (double)m) * inverse);
            const bool near = fabs(left - right) < slack * right && !(exact >> warp & 1);
            verdict = near ? UNSURE : left < right ? ACCEPTED : REJECTED;  // NaN: rejected
          }
        }
      }
      if (lane == 0) {
        sh.row_top[warp] = m;
        sh.row_at[warp] = at;
        sh.row_verdict[warp] = verdict;
      }
    }
    __syncthreads();
    bool again = false;
    for (int r = 0; r < at_once && !stop; ++r) {
      if (sh.row_at[r] == INT_MAX && !(unmasked >> r & 1)) {
        unmasked |= 1u << r;  // the mask allows nothing: all ids
        again = true;
        break;
      }
      const Verdict verdict = sh.row_verdict[r];
      if (!GREEDY && verdict == UNSURE) {
        exact |= 1u << r;
        again = true;
        break;
      }
      top = sh.row_top[r];
      best = sh.row_at[r];
      stop = top == -INFINITY || verdict != ACCEPTED;
      if (!stop) ++kept;
    }
    // the other set next: a slower CTA may still read this one
    turn ^= 1;
    redo = again;
    if (again) {
      kept = i0;  // the round once more, with that row unmasked or exact
    } else if (!stop) {
      i0 += at_once;
      unmasked = exact = 0;
    } else {
      unmasked = unmasked >> (kept - i0) & 1;
    }
  }

  uint32_t* out = v.tokens + (size_t)s * (v.drafts + 1);
  if (rank == 0) {
    for (int i = tid; i <= v.drafts; i += (WARPS * 32)) {
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
  const int run = (hi - lo + WARPS - 1) / WARPS;
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
  // No weight is below e^-670 of the largest: -inf, NaN and what is not allowed
  // come to that too, and shares up to GHOST count as none. Where the logits are
  // so large that their neighbours are further apart, only the largest counts.
  const float lowest = fmaxf(fminf(__fadd_ru(top, -__fmul_rd(670.0f, v.temperature)), __fadd_rd(top, -1e-45f)), -FLT_MAX);
  Draw draw;
  draw.table = sh.table + (lane & (EXP_COPIES - 1));
  draw.lowest = lowest;
  draw.top = top;
  draw.lift = 0.0;
  draw.scale = fmin(inverse * (EXP_ENTRIES * 1.44269504088896340736), -FLOOR / ((double)top - (double)lowest));
  draw.offset = -(double)top * draw.scale;
  // also where the largest logit is the lowest f32 or the largest: -inf, or +inf, needs a look of its own
  const bool edge = fabs(draw.offset) > 0x1p30;
  const int whole_end = row.allowed || edge ? 0 : row.whole_end();  // pieces [1, whole_end) are whole and all allowed
  auto fetch = [&](int c, bool less, Piece<N>& x) {
    const int e0 = row.start(c);
    if (c > 0 && c < whole_end) {
      x.w = *reinterpret_cast<const uint4*>(row.p + e0);
      x.bits = (1u << N) - 1;
    } else {
      x.w = row.raw(c);
      x.bits = row.live(c);
    }
    if (less) {
      if (q && e0 >= 4 && e0 + N + 4 <= v.vocab) {
        // 16-byte loads around the piece; where it starts within them is the same for all pieces of the row
        const float* at = q + e0;
        const int shift = (int)(reinterpret_cast<uintptr_t>(at) / 4 % 4);
        const float4* wide = reinterpret_cast<const float4*>(at - shift);
        float f[N + 4];
#pragma unroll
        for (int k = 0; k < N / 4; ++k) *reinterpret_cast<float4*>(f + 4 * k) = wide[k];
        if (shift) *reinterpret_cast<float4*>(f + N) = wide[N / 4];
        if (shift == 0) {
#pragma unroll
          for (int e = 0; e < N; ++e) x.q[e] = f[e];
        } else if (shift == 1) {
#pragma unroll
          for (int e = 0; e < N; ++e) x.q[e] = f[e + 1];
        } else if (shift == 2) {
#pragma unroll
          for (int e = 0; e < N; ++e) x.q[e] = f[e + 2];
        } else {
#pragma unroll
          for (int e = 0; e < N; ++e) x.q[e] = f[e + 3];
        }
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e) x.q[e] = q && e0 + e >= 0 && e0 + e < v.vocab ? q[e0 + e] : e0 + e == certain ? 1.0f : 0.0f;
      }
    }
  };
  const auto shares = [&](const Piece<N>& p, bool less, double (&x)[N]) {
    if (p.bits == (1u << N) - 1 && !edge) {
      if (less)
        piece_shares<T, true, true>(p, draw, x);
      else
        piece_shares<T, false, true>(p, draw, x);
    } else {
      if (less)
        piece_shares<T, true, false>(p, draw, x);
      else
        piece_shares<T, false, false>(p, draw, x);
    }
  };
  // a run is gone through 32 pieces a step, its steps in DRAW_GROUPS groups
  const int steps = (run + 31) / 32, group = (steps + DRAW_GROUPS - 1) / DRAW_GROUPS * 32;
  auto all_sums = [&](bool less) {  // sh.group[turn] and, in every CTA, sh.draw[turn] = every warp's sum
    double whole = 0.0;
    Piece<N> next;
    if (from + lane < to) fetch(from + lane, less, next);
    for (int g = 0, g0 = from; g < DRAW_GROUPS && g0 < to; ++g, g0 += group) {
      double mine = 0.0;
      for (int c = g0 + lane; c < min(to, g0 + group); c += 32) {
        const Piece<N> now = next;
        if (c + 32 < to) fetch(c + 32, less, next);
        double x[N];
        shares(now, less, x);
#pragma unroll
        for (int e = 0; e < N; e += 2) mine += x[e] + x[e + 1];
      }
      mine = warp_sum(mine);
      if (lane == 0) sh.group[turn][warp][g] = mine;
      whole += mine;
    }
    __syncwarp();
    if (lane < ranks) *cluster.map_shared_rank(&sh.draw[turn][rank * WARPS + warp], lane) = whole;
    cluster.sync();
  };
  const int count = ranks * WARPS;
  auto sum_up = [&] {
    double x = 0.0;
    for (int k = lane; k < count; k += 32) x += sh.draw[turn][k];
    return warp_sum(x);
  };
  all_sums(false);
  double whole = sum_up();
  if (residual) {
    draw.lift = -(double)EXP_ENTRIES * log2(whole);
    draw.offset += draw.lift;
    const int first = turn;
    turn ^= 1;
    all_sums(true);
    const double left = sum_up();
    if (left > GHOSTS) {
      whole = left;
    } else {
      residual = false;  // p nowhere exceeds q: from p
      draw.offset -= draw.lift;
      draw.lift = 0.0;
      turn = first;
    }
  }
  double goal = (double)v.sample[s] * whole;
  goal = goal < GHOSTS ? GHOSTS : goal;  // what counts as none is never drawn; a NaN stays
  // the first warp whose running sum passes the goal; 4 neighbouring sums a lane
  double own[4], upto = 0.0;
  int last = -1;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    own[k] = lane * 4 + k < count ? sh.draw[turn][lane * 4 + k] : 0.0;
    if (own[k] > GHOSTS) last = lane * 4 + k;
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
    if (owner == INT_MAX && own[k] > GHOSTS && ahead + own[k] > goal) {
      owner = lane * 4 + k;
      at_owner = ahead;
    }
    ahead += own[k];
  }
  const int chosen = __reduce_min_sync(FULL, owner);
  const bool end = chosen == INT_MAX;  // a uniform at the very end, or out of range: the last id with a share
  const int winner = end ? __reduce_max_sync(FULL, last) : chosen;
  before = __shfl_sync(FULL, at_owner, (winner >> 2) & 31);
  if (winner == rank * WARPS + warp) {
    // the group first (the last one with a share where the goal is not passed), then the id
    int g = -1;
    {
      double ahead = before;
      for (int k = 0, g0 = from; k < DRAW_GROUPS && g0 < to; ++k, g0 += group) {
        const double x = sh.group[turn][warp][k];
        if (x > GHOSTS) g = k, before = ahead;
        if (x > GHOSTS && ahead + x > goal && !end) break;
        ahead += x;
      }
    }
    int found = -1, final = -1;
    const int g_from = from + max(g, 0) * group, g_to = min(to, g_from + group);
    for (int c0 = g_from; c0 < g_to && found < 0; c0 += 32) {
      const int c = c0 + lane;
      double x[N], mine = 0.0;
      if (c < g_to) {
        Piece<N> p;
        fetch(c, residual, p);
        shares(p, residual, x);
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
      if (c < g_to) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          reach += x[e];
          if (x[e] > GHOST) {
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
    // the order of summing may leave the border a rounding beyond the group's last id
    if (lane == 0) out[kept] = (uint32_t)(found >= 0 ? found : final);
  }
  cluster.sync();
}

template <typename T>
static cudaError_t verify_launch(const VerifyDev& v, int ranks, int warps, int at_once, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(v.sequences * ranks));
  cfg.blockDim = dim3((unsigned)(warps * 32));
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  // a CTA's pieces over a row's threads, 4 pieces a batch at least, and the row's two ends
  const double slack = sum_slack((LogitRow<T>::pieces(v.vocab) / ranks + 1) / (warps / at_once * 32 * 4) + 4);
  if (v.temperature == 0.0f) return cudaLaunchKernelEx(&cfg, warps == 16 ? k_verify<T, true, 16> : k_verify<T, true, 8>, v, at_once, slack);
  return cudaLaunchKernelEx(&cfg, warps == 16 ? k_verify<T, false, 16> : k_verify<T, false, 8>, v, at_once, slack);
}

cudaError_t verify_drafts(const VerifyDev& v, cudaStream_t st) {
  if (v.sequences == 0) return cudaSuccess;
  const int size = v.dtype == DTYPE_F32 ? 4 : 2;
  // About 480 CTAs of 8 warps, up to 8 for a sequence (96 rows of 129283: 5 CTAs
  // 95 us, 4 101, 2 154, 8 115; 256 of 8192: 2 CTAs 36 us, 1 40, 4 47); where
  // that leaves SMs empty, of 16 warps.
  const int n = v.sequences;
  int ranks = (480 + n / 2) / n, warps = 8;
  ranks = ranks < 1 ? 1 : ranks > VERIFY_MAX_CLUSTER ? VERIFY_MAX_CLUSTER : ranks;
  if (n * ranks <= 148) warps = 16;
  // Rows of a round: two, or more where a CTA's slices of them are 16 KB at
  // most (one sequence of 8192: 4 rows 12.5 us, 2 16.1; a row read in vain
  // costs less than a round of its own); four at temperature 0, where a row is
  // only looked through for its maximum (200 of 50257 in 16 bits: 4 rows 40 us,
  // 2 46; 96 of 129283 at temperature 1: 104 and 99).
  const long long slice = (long long)v.vocab * size / ranks;
  int at_once = 1;
  const int least = v.temperature == 0.0f ? 4 : 2;
  while (at_once < VERIFY_MAX_ROWS && at_once < v.drafts + 1 && (at_once < least || slice * at_once < 16384)) at_once *= 2;
  if (v.dtype == DTYPE_F32) return verify_launch<float>(v, ranks, warps, at_once, st);
  if (v.dtype == DTYPE_F16) return verify_launch<__half>(v, ranks, warps, at_once, st);
  return verify_launch<__nv_bfloat16>(v, ranks, warps, at_once, st);
}

}  // namespace nbk
