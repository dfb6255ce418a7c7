// label_probs.hip — what a row of logits says, and learning from it: label log probabilities with entropy and the best
// alternatives (forward, backward), and the divergence of a teacher's top logits (forward, backward).
//
// Mathematics.  Row x of V logits, c = log2(e) / tau (tau = 1 for the label statistics).  With a reference M2 = fl(m c),
// m the running maximum, one pass keeps
//     s  = sum 2^(x c - M2)          se = sum 2^(x c - M2) (x c - M2)          (x c - M2: one FMA, one rounding)
// and moves both to a new reference M2' by  f = 2^(M2 - M2'):  se <- (se + s (M2 - M2')) f,  s <- s f.
// ls2 = log2(s) - (m c - M2) is the row's log2-sum-exp relative to its maximum, hence
//     log p_v = ((x_v - m) c - ls2) ln 2,   H = (log2(s) - se / s) ln 2,   p_v = 2^((x_v - m) c - ls2).
// m, s, se are fp32 whatever the logits' type; only d logits is rounded to it, once.
//     d x_v = g ([v = y] - p_v) - h p_v (log p_v + H)                      (label: g, h = gradients of log p_y and H)
//     d x_v = g tau (p_v - sum_j q_j [i_j = v]),  loss = tau^2 sum_j q_j (log q_j - log p_{i_j})   (q: softmax of the teacher's k)
//
// Masked entries are logits of -inf: probability 0, never an alternative, gradient 0 from the p terms.  The type's lowest
// finite value is an ordinary logit (a row of nothing else is uniform): rows whose |maximum| c passes 1e37, where x c can
// overflow, are summed again with (x - m) c.
//
// Alternatives without a compare per element: every thread keeps the key (maximum, first vector that holds it) of its share
// of the row.  64 groups of threads give 64 distinct keys; the k-th best of them is a lower bound of the k best elements (k groups
// hold one at least as good), so only the shares of threads whose key reaches it are looked at again (from L2): for k = 20 about
// 24 of 512.  Their elements at or above the bound are ranked by counting.
#include "head_common.h"

namespace {

constexpr int kMaxTop = 64;              // one alternative per lane, one group of threads per alternative
constexpr int kSmallV = 2048;            // up to here: one wave per row, the row in registers

// order-preserving map float -> unsigned (-0 = +0; -inf -> kKeyNegInf; 0 = "nothing")
constexpr unsigned kKeyNegInf = 0x007fffffu;
__device__ __forceinline__ unsigned lp_key(float v) {
  const unsigned b = __builtin_bit_cast(unsigned, v + 0.f);
  return (int)b < 0 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float lp_unkey(unsigned k) {
  return __builtin_bit_cast(float, (int)k < 0 ? k & 0x7fffffffu : ~k);
}

// how many of the first n lanes' keys are larger than this lane's (equal keys: only 0, "nothing")
__device__ __forceinline__ int lp_rank64(u64 key, int n) {
  int rank = 0;
  if (n >= 64) {
#pragma unroll 8
    for (int q = 0; q < 64; ++q) rank += pn2_readlane_u64(key, q) > key ? 1 : 0;
  } else {
    for (int q = 0; q < n; ++q) rank += pn2_readlane_u64(key, q) > key ? 1 : 0;
  }
  return rank;
}

struct RowSum {          // running statistics of (a part of) a row
  float m, M2, s, se;
};
struct RowStat {         // ... of a whole row: ls2 = log2 sum 2^((x - m) c), -inf for a row of nothing but -inf; entropy in nats
  float m, ls2, entropy;
  bool empty, nan;
};

// c scales logits to log2 units; |m| <= lim keeps m c far from overflow
__device__ __forceinline__ float lp_lim(float c) { return 1e37f / fmaxf(c, 1.f); }
__device__ __forceinline__ float lp_ref(float m, float c, float lim) { return fmaxf(m, -lim) * c; }

// add n values (all of one batch) whose maximum is bm
template <bool ENT, int N>
__device__ __forceinline__ void lp_add(RowSum &r, const float (&x)[N], float bm, float c, float lim) {
  const float nm = fmaxf(r.m, bm);
  const float M2 = lp_ref(nm, c, lim);
  const float d = r.M2 - M2, f = hd_exp2(d);
  if constexpr (ENT) r.se = __fmaf_rn(r.s, d, r.se) * f;
  r.s *= f;
  r.m = nm;
  r.M2 = M2;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float t = __fmaf_rn(x[i], c, -M2), e = hd_exp2(t);
    r.s += e;
    if constexpr (ENT) r.se = __fmaf_rn(e, fmaxf(t, -1e30f), r.se);      // (0 * -inf of a masked entry counts as 0)
  }
}

// bring a thread's sums to the common maximum m and add them over the wave
template <bool ENT>
__device__ __forceinline__ RowSum lp_wave_combine(RowSum r, float c, float lim) {
  RowSum o;
  o.m = hd_wave_max(r.m);
  o.M2 = lp_ref(o.m, c, lim);
  const float d = r.M2 - o.M2, f = hd_exp2(d);
  o.s = hd_wave_sum(r.s * f);
  o.se = ENT ? hd_wave_sum(__fmaf_rn(r.s, d, r.se) * f) : 0.f;
  return o;
}

// the row's results from its sums, whose reference lies `res` log2 units below m c
__device__ __forceinline__ RowStat lp_stat(const RowSum &r, float res) {
  RowStat o;
  const float l = log2f(r.s);
  o.m = r.m;
  o.empty = r.m == -kHdInf && r.s == 0.f;
  o.nan = !(r.s == r.s);
  o.ls2 = o.empty ? -kHdInf : l - res;
  o.entropy = o.empty ? 0.f : (l - r.se / r.s) * kHdLn2;
  return o;
}
// (temperature 1)
__device__ __forceinline__ float lp_logp(float x, const RowStat &r) { return r.empty ? -kHdInf : __fmaf_rn(-r.ls2, kHdLn2, x - r.m); }

struct FwdArgs {
  long long T, ld;
  int V, top, k;
  float c, tau;
  const void *logits;
  const long long *labels;
  long long ignore;
  float *log_prob, *entropy, *stats;
  float *top_lp;
  long long *top_idx;
  const long long *t_idx;          // distill: the teacher's indices (T, k), values (T, k), loss (T)
  const void *t_val;
  int t_dtype;
  float *loss;
  int nseg, seg;                   // a row in nseg segments of seg entries (the last one shorter): their sums (T, nseg, 4), the keys
  float *part;                     // of threads (T, nseg, 256)
  u64 *keys;
};

__device__ __forceinline__ float lp_teacher(const FwdArgs &a, long long at) {
  if (a.t_dtype == PN2_DT_F32) return ((const float *)a.t_val)[at];
  if (a.t_dtype == PN2_DT_BF16) return (float)((const __bf16 *)a.t_val)[at];
  return (float)((const _Float16 *)a.t_val)[at];
}

// A row's label and its logit, read before the row itself (two dependent round trips to memory).
struct Label {
  long long y;
  float x;
};
template <class T>
__device__ __forceinline__ Label lp_label(const FwdArgs &a, long long row, const typename T::elem *x) {
  Label l;
  l.y = a.labels[row];
  l.x = l.y >= 0 && l.y < a.V ? T::load(x + l.y) : __builtin_nanf("");
  return l;
}
// One wave finishes a label row: stats are wave-uniform.
__device__ __forceinline__ void lp_finish_label(const FwdArgs &a, long long row, const Label &l, const RowStat &r) {
  if (pn2_lane() == 0) {
    float lp = 0.f;
    if (l.y != a.ignore) lp = l.y < 0 || l.y >= a.V ? l.x : lp_logp(l.x, r);
    a.log_prob[row] = lp;
    a.entropy[row] = r.entropy;
    if (a.stats) {
      a.stats[2 * row] = r.m;
      a.stats[2 * row + 1] = r.ls2;
    }
  }
}

// One wave finishes a distillation row.  An unused slot has a negative index or the value -inf; a row without a used slot
// has no loss (and its logits were not read: r is not looked at).  An index >= V of a used slot makes the row NaN.
__device__ __forceinline__ bool lp_teacher_any(const FwdArgs &a, long long row) {
  bool any = false;
  for (int j = pn2_lane(); j < a.k; j += PN2_WAVE)
    any |= a.t_idx[row * a.k + j] >= 0 && !(lp_teacher(a, row * a.k + j) == -kHdInf);
  return __ballot(any) != 0;
}
template <class T>
__device__ __forceinline__ void lp_finish_distill(const FwdArgs &a, long long row, const typename T::elem *x, const RowStat &r,
                                                  bool any) {
  const int lane = pn2_lane();
  if (!any) {
    if (lane == 0) {
      a.loss[row] = 0.f;
      if (a.stats) {
        a.stats[4 * row] = a.stats[4 * row + 2] = -kHdInf;
        a.stats[4 * row + 1] = a.stats[4 * row + 3] = 0.f;
      }
    }
    return;
  }
  const long long at = row * a.k;
  float tm = -kHdInf;
  bool bad = false;
  for (int j = lane; j < a.k; j += PN2_WAVE) {
    const long long i = a.t_idx[at + j];
    const float t = lp_teacher(a, at + j);
    if (i >= 0) tm = fmaxf(tm, t);
    bad |= i >= a.V && !(t == -kHdInf);
  }
  tm = hd_wave_max(tm);
  bad = __ballot(bad) != 0;
  float ts = 0.f;
  for (int j = lane; j < a.k; j += PN2_WAVE)
    if (a.t_idx[at + j] >= 0) ts += hd_exp2((lp_teacher(a, at + j) - tm) * a.c);
  ts = hd_wave_sum(ts);
  const float tls2 = log2f(ts);
  const float ls2 = bad ? __builtin_nanf("") : r.ls2;
  float acc = 0.f;
  if (!bad)
    for (int j = lane; j < a.k; j += PN2_WAVE) {
      const long long i = a.t_idx[at + j];
      if (i < 0) continue;
      const float lq2 = (lp_teacher(a, at + j) - tm) * a.c - tls2, q = hd_exp2(lq2);
      if (q == 0.f) continue;
      acc += r.empty ? kHdInf : q * ((lq2 - ((T::load(x + i) - r.m) * a.c - ls2)) * kHdLn2);
    }
  acc = hd_wave_sum(acc);
  if (lane == 0) {
    a.loss[row] = bad ? __builtin_nanf("") : acc * a.tau * a.tau;
    if (a.stats) {
      a.stats[4 * row] = r.m;
      a.stats[4 * row + 1] = ls2;
      a.stats[4 * row + 2] = tm;
      a.stats[4 * row + 3] = tls2;
    }
  }
}

enum { MODE_LABEL, MODE_DISTILL };

// alternative `slot` of a row, should no entry take it
__device__ __forceinline__ void lp_clear(const FwdArgs &a, long long row, int slot, const RowStat &st) {
  a.top_lp[row * a.top + slot] = st.nan ? __builtin_nanf("") : -kHdInf;
  a.top_idx[row * a.top + slot] = -1;
}

// one of the n candidates in LDS takes the place its rank gives it
__device__ __forceinline__ void lp_place(const FwdArgs &a, long long row, const u64 *cand, int n, u64 mine, const RowStat &st) {
  int rank = 0;
#pragma unroll 8
  for (int q = 0; q < n; ++q) rank += cand[q] > mine ? 1 : 0;
  if (rank < a.top) {
    a.top_lp[row * a.top + rank] = lp_logp(lp_unkey((unsigned)(mine >> 32)), st);
    a.top_idx[row * a.top + rank] = (int)~(unsigned)mine;
  }
}

// ------------------------------------------------------------------------------------------------ V <= 2048: a wave per row
template <class T, int MODE, int EPL>
__global__ __launch_bounds__(256) void lp_small_kernel(FwdArgs a) {
  const long long row = hd_block() * 4 + (threadIdx.x >> 6);
  if (row >= a.T) return;
  const int lane = pn2_lane();
  const typename T::elem *x = (const typename T::elem *)a.logits + row * a.ld;
  RowSum r{-kHdInf, 0.f, 0.f, 0.f};
  if constexpr (MODE == MODE_DISTILL) {
    if (!lp_teacher_any(a, row)) {
      lp_finish_distill<T>(a, row, x, RowStat{}, false);
      return;
    }
  }
  Label label{};
  if constexpr (MODE == MODE_LABEL) label = lp_label<T>(a, row, x);
  float v[EPL];
  float m = -kHdInf;
#pragma unroll
  for (int j = 0; j < EPL; ++j) {                      // (loads at clamped places: a branch each would make them wait for each other)
    const int i = lane + j * PN2_WAVE;
    v[j] = T::load(x + (i < a.V ? i : a.V - 1));
  }
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    v[j] = lane + j * PN2_WAVE < a.V ? v[j] : -kHdInf;
    m = fmaxf(m, v[j]);
  }
  // the maximum is known before the sum: exact differences, no limits needed
  r.m = hd_wave_max(m);
  float s = 0.f, se = 0.f;
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    // (an entry of -inf adds nothing; of an empty row, x - m would be NaN)
    const float t = (v[j] - r.m) * a.c, e = v[j] == -kHdInf ? 0.f : hd_exp2(t);
    s += e;
    if constexpr (MODE == MODE_LABEL) se += v[j] == -kHdInf ? 0.f : e * fmaxf(t, -1e30f);
  }
  r.s = hd_wave_sum(s);
  r.se = hd_wave_sum(se);
  const RowStat f = lp_stat(r, 0.f);
  if constexpr (MODE == MODE_DISTILL) {
    lp_finish_distill<T>(a, row, x, f, true);
  } else {
    lp_finish_label(a, row, label, f);
    if (a.top) {
      // the k-th best of the 64 lanes' best keys bounds the k best elements from below; those at or above it are ranked by counting
      __shared__ u64 sh_cand[4][EPL * PN2_WAVE];
      const int w = threadIdx.x >> 6;
      u64 best = 0u;
#pragma unroll
      for (int j = 0; j < EPL; ++j) {
        const unsigned k = lp_key(v[j]);
        const u64 key = k <= kKeyNegInf ? 0u : ((u64)k << 32) | (unsigned)~(lane + j * PN2_WAVE);
        best = key > best ? key : best;
      }
      const int rank = lp_rank64(best, a.V);
      if (lane < a.top) {                              // slots that no entry will take
        a.top_lp[row * a.top + lane] = f.nan ? __builtin_nanf("") : -kHdInf;
        a.top_idx[row * a.top + lane] = -1;
      }
      if (f.nan) return;
      if constexpr (EPL == 1) {                        // the lanes' keys are the elements
        if (best != 0u && rank < a.top) {
          a.top_lp[row * a.top + rank] = lp_logp(v[0], f);
          a.top_idx[row * a.top + rank] = lane;
        }
        return;
      }
      const u64 hit = __ballot(rank == a.top - 1 && best != 0u);
      const u64 low = hit ? pn2_readlane_u64(best, __ffsll((unsigned long long)hit) - 1) : (u64)(kKeyNegInf + 1) << 32;
      int n = 0;
#pragma unroll
      for (int j = 0; j < EPL; ++j) {
        const unsigned k = lp_key(v[j]);
        const u64 key = ((u64)k << 32) | (unsigned)~(lane + j * PN2_WAVE);
        const u64 mask = __ballot(key >= low);
        if (key >= low) sh_cand[w][n + pn2_prefix_popc(mask)] = key;
        n += __popcll(mask);
      }
      __builtin_amdgcn_wave_barrier();                 // (LDS operations of a wave are in order)
      for (int e = lane; e < n; e += PN2_WAVE) lp_place(a, row, sh_cand[w], n, sh_cand[w][e], f);
    }
  }
}

// --------------------------------------------------------------------------------------------- V > 2048: a workgroup per row
constexpr int kCand = 1024;              // elements kept in LDS for the final ranking

// a row (or a segment of one) in vectors of 16 bytes; what lies behind its end reads as -inf
template <class T>
struct Vectors {
  const typename T::elem *x;
  int nfull, tail, nvec;
  __device__ __forceinline__ Vectors(const typename T::elem *x_, int V) : x(x_), nfull(V / T::kPerVec), tail(V % T::kPerVec) {
    nvec = nfull + (tail != 0);
  }
  __device__ __forceinline__ hd_u32x4 nothing() const {
    float g[T::kPerVec];
#pragma unroll
    for (int j = 0; j < T::kPerVec; ++j) g[j] = -kHdInf;
    return T::pack(g);
  }
  // the last, partial vector
  __device__ __forceinline__ hd_u32x4 last() const {
    float g[T::kPerVec];
#pragma unroll
    for (int j = 0; j < T::kPerVec; ++j) g[j] = j < tail ? T::load(x + (long long)nfull * T::kPerVec + j) : -kHdInf;
    return T::pack(g);
  }
  // vector i if it is a whole one.  (A load at a clamped place and a choice: no branch in front of the loads.)
  __device__ __forceinline__ hd_u32x4 whole(int i) const {
    const hd_u32x4 w = hd_load16<T>(x + (long long)(i < nfull ? i : nfull - 1) * T::kPerVec);
    return i < nfull ? w : nothing();
  }
  __device__ __forceinline__ hd_u32x4 fetch(int i) const {
    hd_u32x4 w = whole(i);
    if (tail && i == nfull) w = last();
    return w;
  }
};

// The alternatives of a row by a whole workgroup: `mine` is the best key of a thread's share of shares, winners(low, push) names its
// shares whose key reaches `low` (WIN in all at most), share(w) says where one lies: every STRIDE-th vector of a stretch.
struct Share {
  int first, end;
};
template <class T, int BT, int STRIDE, int WIN, class Winners, class ShareOf>
__device__ __forceinline__ void lp_select(const FwdArgs &a, long long row, const Vectors<T> &v, const RowStat &st, u64 mine, Winners winners,
                                          ShareOf share) {
  constexpr int VE = T::kPerVec, W = BT / PN2_WAVE;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  __shared__ u64 sh_group[64], sh_low;
  __shared__ int sh_win[WIN], sh_count[2];            // winners, candidates
  __shared__ u64 sh_cand[kCand + 1], sh_best[W];
  // the best key of each of 64 groups of neighbouring threads; the k-th best of them bounds the k best elements from below
  u64 g = mine;
  {
    u64 o = pn2_dpp_u64<PN2_DPP_QUAD_XOR1>(g);
    g = o > g ? o : g;
    o = pn2_dpp_u64<PN2_DPP_QUAD_XOR2>(g);
    g = o > g ? o : g;
    if constexpr (BT >= 512) { o = pn2_dpp_u64<PN2_DPP_ROW_HALF_MIRROR>(g); g = o > g ? o : g; }
    if constexpr (BT >= 1024) { o = pn2_dpp_u64<PN2_DPP_ROW_MIRROR>(g); g = o > g ? o : g; }
  }
  if (tid % (BT / 64) == 0) sh_group[tid / (BT / 64)] = g;
  if (tid < 2) sh_count[tid] = 0;
  if (tid < a.top) lp_clear(a, row, tid, st);
  __syncthreads();
  if (st.nan) return;                                // uniform over the workgroup
  if (wave == 0) {
    const u64 k = sh_group[lane];
    const int rank = lp_rank64(k, 64);               // (keys of non-empty groups differ: their vectors do)
    const u64 hit = __ballot(rank == a.top - 1 && k != 0u);
    const u64 low = hit ? pn2_readlane_u64(k, __ffsll((unsigned long long)hit) - 1) : (u64)(kKeyNegInf + 1) << 32;
    if (lane == 0) sh_low = low;
  }
  __syncthreads();
  const u64 low = sh_low;
  winners(low, [&](int w) { sh_win[atomicAdd(&sh_count[0], 1)] = w; });        // (any order: the ranking below is total)
  __syncthreads();
  const int nwin = sh_count[0];
  // (one share at a time: a single row's time is this code's trip through the instruction cache, 15.1 us against 16.5 us unrolled)
  for (int w = wave; w < nwin; w += W) {
    const Share s = share(sh_win[w]);
    for (int i = s.first + lane * STRIDE; __builtin_amdgcn_readfirstlane(i) < s.end; i += STRIDE * PN2_WAVE) {   // its vectors, one per lane
      float f[VE];
      T::unpack(i < s.end ? v.fetch(i) : v.nothing(), f);
      unsigned k[VE], hits = 0u;
#pragma unroll
      for (int j = 0; j < VE; ++j) {
        k[j] = lp_key(f[j]);
        // (what lies behind the row's end reads as -inf, below any bound)
        if ((((u64)k[j] << 32) | (unsigned)~i) >= low) hits |= 1u << j;
      }
      if (hits) {
        const int at = atomicAdd(&sh_count[1], __popc(hits));
#pragma unroll
        for (int j = 0; j < VE; ++j) {               // (what is no candidate, or one too many, goes to a slot that nobody reads)
          const int to = at + __popc(hits & ((1u << j) - 1u));
          sh_cand[((hits >> j) & 1u) && to < kCand ? to : kCand] = ((u64)k[j] << 32) | (unsigned)~(i * VE + j);
        }
      }
    }
  }
  __syncthreads();
  const int n = sh_count[1];
  if (n <= kCand) {
    for (int e = tid; e < n; e += BT) lp_place(a, row, sh_cand, n, sh_cand[e], st);
    return;
  }
  // rows with very many equal entries at the bound: one pass over the row per alternative, each the best below the last
  u64 last = ~(u64)0;
  for (int q = 0; q < a.top; ++q) {
    u64 best = 0u;
    for (int i = tid; i < v.nvec; i += BT) {
      float f[VE];
      T::unpack(v.fetch(i), f);
#pragma unroll
      for (int j = 0; j < VE; ++j) {
        const unsigned k = lp_key(f[j]);
        const u64 key = ((u64)k << 32) | (unsigned)~(i * VE + j);
        if (k > kKeyNegInf && key < last && key > best) best = key;
      }
    }
    best = pn2_wave_max_u64(best);
    if (lane == 0) sh_best[wave] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; ++w) best = sh_best[w] > best ? sh_best[w] : best;
    __syncthreads();
    if (best == 0u) break;                           // uniform over the workgroup
    if (tid == 0) {
      a.top_lp[row * a.top + q] = lp_logp(lp_unkey((unsigned)(best >> 32)), st);
      a.top_idx[row * a.top + q] = (int)~(unsigned)best;
    }
    last = best;
  }
}

// (x - m) c summed again where x c may overflow; by the whole workgroup, behind a barrier
template <class T, bool ENT, int BT>
__device__ __forceinline__ void lp_sum_again(RowSum &r, const typename T::elem *x, int V, float c, float *sh_s, float *sh_se) {
  constexpr int W = BT / PN2_WAVE;
  float s = 0.f, se = 0.f;
  for (int i = threadIdx.x; i < V; i += BT) {
    const float t = (T::load(x + i) - r.m) * c, e = hd_exp2(t);
    s += e;
    if constexpr (ENT) se += e * fmaxf(t, -1e30f);
  }
  s = hd_wave_sum(s);
  se = hd_wave_sum(se);
  __syncthreads();
  if (pn2_lane() == 0) { sh_s[threadIdx.x >> 6] = s; sh_se[threadIdx.x >> 6] = se; }
  __syncthreads();
  r.s = r.se = 0.f;
#pragma unroll
  for (int w = 0; w < W; ++w) { r.s += sh_s[w]; r.se += sh_se[w]; }
}

// SEG: a workgroup per segment of a row instead, which leaves its sums and its best entries' keys for lp_join_kernel.
template <class T, int MODE, bool TOP, int BT, int U, bool SEG>
__global__ __launch_bounds__(BT) void lp_row_kernel(FwdArgs a) {
  constexpr int VE = T::kPerVec, W = BT / PN2_WAVE;
  constexpr bool ENT = MODE == MODE_LABEL;
  typedef typename T::elem elem;
  __shared__ float sh_m[W], sh_s[W], sh_se[W];
  const long long unit = hd_block(), row = SEG ? unit / a.nseg : unit;
  if (row >= a.T) return;
  const int from = SEG ? (int)(unit - row * a.nseg) * a.seg : 0, V = SEG ? (a.V - from < a.seg ? a.V - from : a.seg) : a.V;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const elem *x = (const elem *)a.logits + row * a.ld + from;
  RowSum r{-kHdInf, 0.f, 0.f, 0.f};
  if constexpr (MODE == MODE_DISTILL) {
    if (!lp_teacher_any(a, row)) {                     // the same answer in every wave
      if (!SEG && wave == 0) lp_finish_distill<T>(a, row, x, RowStat{}, false);
      return;
    }
  }
  Label label{};
  if constexpr (MODE == MODE_LABEL && !SEG) {
    if (wave == W - 1) label = lp_label<T>(a, row, x);
  }
  const float c = a.c, lim = lp_lim(c);
  r.M2 = lp_ref(r.m, c, lim);
  // (Vectors written out: as a class here, its loads are scheduled worse, 1021 x 50021 fp16 23.7 us instead of 23.0)
  const int nfull = V / VE, tail = V % VE;
  int ord = 0x7fffffff;                                // first vector that holds the thread's maximum
  auto last_vector = [&]() -> hd_u32x4 {
    float g[VE];
#pragma unroll
    for (int j = 0; j < VE; ++j) g[j] = j < tail ? T::load(x + (long long)nfull * VE + j) : -kHdInf;
    return T::pack(g);
  };
  hd_u32x4 nothing;
  {
    float g[VE];
#pragma unroll
    for (int j = 0; j < VE; ++j) g[j] = -kHdInf;
    nothing = T::pack(g);
  }
  auto whole = [&](int i) -> hd_u32x4 {
    const hd_u32x4 w = hd_load16<T>(x + (long long)(i < nfull ? i : nfull - 1) * VE);
    return i < nfull ? w : nothing;
  };
  hd_u32x4 behind = nothing;
  if (tail && tid == nfull % BT) behind = last_vector();
  for (int b = 0; b < nfull; b += BT * U) {
    hd_u32x4 w[U];
    if (b + BT * U <= nfull) {
#pragma unroll
      for (int u = 0; u < U; ++u) w[u] = hd_load16<T>(x + (long long)(b + u * BT + tid) * VE);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) w[u] = whole(b + u * BT + tid);
    }
    float f[U * VE];
    float bm = -kHdInf;
    float best = r.m;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float g[VE];
      T::unpack(w[u], g);
      float vm = g[0];
#pragma unroll
      for (int i = 0; i < VE; ++i) { f[u * VE + i] = g[i]; vm = fmaxf(vm, g[i]); }
      if constexpr (TOP) {
        if (vm > best) { best = vm; ord = b + u * BT + tid; }
      }
      bm = fmaxf(bm, vm);
    }
    lp_add<ENT>(r, f, bm, c, lim);
  }
  if (tail) {
    float f[VE];
    T::unpack(behind, f);
    float vm = f[0];
#pragma unroll
    for (int i = 1; i < VE; ++i) vm = fmaxf(vm, f[i]);
    if constexpr (TOP) {
      if (vm > r.m) ord = nfull;
    }
    lp_add<ENT>(r, f, vm, c, lim);
  }
  const float own = r.m;
  // the row's sums, in a fixed order
  {
    const RowSum o = lp_wave_combine<ENT>(r, c, lim);
    if (lane == 0) { sh_m[wave] = o.m; sh_s[wave] = o.s; sh_se[wave] = o.se; }
    __syncthreads();
    r.m = sh_m[0];
#pragma unroll
    for (int w = 1; w < W; ++w) r.m = fmaxf(r.m, sh_m[w]);
    r.M2 = lp_ref(r.m, c, lim);
    r.s = r.se = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float d = lp_ref(sh_m[w], c, lim) - r.M2, f = hd_exp2(d);
      r.s = __fmaf_rn(sh_s[w], f, r.s);
      if constexpr (ENT) r.se = __fmaf_rn(__fmaf_rn(sh_s[w], d, sh_se[w]), f, r.se);
    }
  }
  RowStat st{};
  if constexpr (SEG) {
    if (tid == 0) hd_store16<HdF32>(a.part + unit * 4, HdF32::pack({r.m, r.s, r.se, 0.f}));
  } else {
    float res = __fmaf_rn(r.m, c, -r.M2);
    if (fabsf(r.m) > lim && fabsf(r.m) < kHdInf) {     // uniform over the workgroup; every wave has passed the barrier above
      lp_sum_again<T, ENT, BT>(r, x, V, c, sh_s, sh_se);
      res = 0.f;
    }
    st = lp_stat(r, res);
    if constexpr (MODE == MODE_DISTILL) {
      if (wave == 0) lp_finish_distill<T>(a, row, x, st, true);
      return;
    }
    if (wave == W - 1) lp_finish_label(a, row, label, st);
  }
  if constexpr (TOP) {
    // keys as one number: value above, vector below, earlier ones larger
    const u64 mine = own == -kHdInf ? 0u : ((u64)lp_key(own) << 32) | (unsigned)~(ord + (SEG ? from / VE : 0));
    if constexpr (SEG) {
      a.keys[unit * BT + tid] = mine;
    } else {
      const Vectors<T> v(x, V);
      lp_select<T, BT, BT, BT>(
          a, row, v, st, mine,
          [&](u64 low, auto push) { if (mine >= low && mine != 0u) push(tid); },
          [&](int w) { return Share{w, v.nvec}; });
    }
  }
}

// A row's segments joined: their sums by every wave (one segment per lane), then the alternatives, from the keys of the segments' threads.
constexpr int kSegThreads = 256, kMaxSeg = 32;
template <class T, int MODE, bool TOP, int BT>
__global__ __launch_bounds__(BT) void lp_join_kernel(FwdArgs a) {
  constexpr bool ENT = MODE == MODE_LABEL;
  constexpr int W = BT / PN2_WAVE, NK = kMaxSeg * kSegThreads / BT;
  __shared__ float sh_s[W], sh_se[W];
  const long long row = blockIdx.x;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const Vectors<T> v((const typename T::elem *)a.logits + row * a.ld, a.V);
  if constexpr (MODE == MODE_DISTILL) {
    if (!lp_teacher_any(a, row)) {
      if (wave == 0) lp_finish_distill<T>(a, row, v.x, RowStat{}, false);
      return;
    }
  }
  u64 key[TOP ? NK : 1] = {}, mine = 0u;
  if constexpr (TOP) {
#pragma unroll
    for (int q = 0; q < NK; ++q) {                     // (loads at clamped places)
      const int at = q * BT + tid, n = a.nseg * kSegThreads;
      const u64 k = a.keys[row * n + (at < n ? at : 0)];
      key[q] = at < n ? k : 0u;
    }
  }
  const float c = a.c, lim = lp_lim(c);
  float f[4];
  HdF32::unpack(hd_load16<HdF32>(a.part + (row * a.nseg + (lane < a.nseg ? lane : 0)) * 4), f);
  Label label{};
  if constexpr (MODE == MODE_LABEL) {
    if (wave == W - 1) label = lp_label<T>(a, row, v.x);
  }
  const bool on = lane < a.nseg;
  RowSum r{on ? f[0] : -kHdInf, 0.f, on ? f[1] : 0.f, on ? f[2] : 0.f};
  r.M2 = lp_ref(r.m, c, lim);
  r = lp_wave_combine<ENT>(r, c, lim);
  float res = __fmaf_rn(r.m, c, -r.M2);
  if (fabsf(r.m) > lim && fabsf(r.m) < kHdInf) {       // uniform over the workgroup
    lp_sum_again<T, ENT, BT>(r, v.x, a.V, c, sh_s, sh_se);
    res = 0.f;
  }
  const RowStat st = lp_stat(r, res);
  if constexpr (MODE == MODE_DISTILL) {
    if (wave == 0) lp_finish_distill<T>(a, row, v.x, st, true);
    return;
  }
  if (wave == W - 1) lp_finish_label(a, row, label, st);
  if constexpr (TOP) {
#pragma unroll
    for (int q = 0; q < NK; ++q) mine = key[q] > mine ? key[q] : mine;
    const int each = a.seg / T::kPerVec;
    lp_select<T, BT, kSegThreads, kMaxSeg * kSegThreads>(
        a, row, v, st, mine,
        [&](u64 low, auto push) {
#pragma unroll
          for (int q = 0; q < NK; ++q)
            if (key[q] >= low && key[q] != 0u) push(q * BT + tid);
        },
        [&](int w) {
          const int seg = w / kSegThreads, end = (seg + 1) * each;
          return Share{seg * each + w % kSegThreads, end < v.nvec ? end : v.nvec};
        });
  }
}

// ------------------------------------------------------------------------------------------------------------- backward
struct BwdArgs {
  long long T, ld;
  int V, k, nseg;
  float c, tau;
  const void *logits;
  const long long *labels;
  long long ignore;
  const float *stats, *entropy, *g_lp, *g_ent;      // g_lp / g_ent / g_loss: NULL = zero
  const long long *t_idx;
  const void *t_val;
  int t_dtype;
  const float *g_loss;
  void *dlogits;
};

__device__ __forceinline__ float lp_teacher(const BwdArgs &a, long long at) {
  if (a.t_dtype == PN2_DT_F32) return ((const float *)a.t_val)[at];
  if (a.t_dtype == PN2_DT_BF16) return (float)((const __bf16 *)a.t_val)[at];
  return (float)((const _Float16 *)a.t_val)[at];
}

constexpr int kTeacher = 256;            // a teacher's indices kept in LDS; further ones are read again

// GROUP threads own a segment of one row.  Bound by its bytes (V read, V written); ~6 vector instructions per element.
template <class T, int MODE, int GROUP>
__global__ __launch_bounds__(256) void lp_grad_kernel(BwdArgs a) {
  constexpr int VE = T::kPerVec, U = 4;
  typedef typename T::elem elem;
  const int tid = threadIdx.x % GROUP;
  const long long unit = GROUP == 256 ? hd_block() : hd_block() * (256 / GROUP) + threadIdx.x / GROUP;
  const long long nth = unit / a.nseg;
  if (nth >= a.T) return;                              // (a whole workgroup, or GROUP < 256: no barrier below is left behind)
  const long long row = a.T - 1 - nth;                 // the rows the forward pass read last may still be in the cache
  const int seg = (int)(unit - nth * a.nseg);
  const elem *x = (const elem *)a.logits + row * a.ld;
  elem *dx = (elem *)a.dlogits + row * (long long)a.V;
  const int nfull = a.V / VE, tail = a.V % VE, nvec = nfull + (tail != 0);
  const int v0 = seg * GROUP * U, v1 = v0 + GROUP * U < nvec ? v0 + GROUP * U : nvec;

  const float c = a.c;
  float m, ls2, A = 0.f, Bc = 0.f, H = 0.f, g1 = 0.f;
  long long y = -1;
  bool zero;
  if constexpr (MODE == MODE_LABEL) {
    m = a.stats[2 * row];
    ls2 = a.stats[2 * row + 1];
    y = a.labels[row];
    const bool skip = y == a.ignore;
    g1 = a.g_lp && !skip ? a.g_lp[row] : 0.f;
    const float h = a.g_ent ? a.g_ent[row] : 0.f;
    if (!skip && (y < 0 || y >= a.V)) { if (a.g_lp) g1 = __builtin_nanf(""); y = -1; }
    if (skip) y = -1;
    H = a.entropy[row];
    A = -(g1 + h * H);                                 // d x_v = p_v (A + Bc ln p2_v) + [v = y] g1
    Bc = -h * kHdLn2;
    zero = (m == -kHdInf && ls2 == -kHdInf) || (g1 == 0.f && h == 0.f);
  } else {
    m = a.stats[4 * row];
    ls2 = a.stats[4 * row + 1];
    g1 = a.g_loss ? a.g_loss[row] * a.tau : 0.f;
    A = g1;
    zero = a.stats[4 * row + 2] == -kHdInf || (m == -kHdInf && ls2 == -kHdInf) || g1 == 0.f;
  }
  // gradient of one entry without the label / teacher term
  auto grad = [&](float xv) -> float {
    const float t = __fmaf_rn(xv - m, c, -ls2), p = hd_exp2(t);
    if constexpr (MODE == MODE_LABEL) {
      const float w = __fmaf_rn(Bc, fmaxf(t, -1e30f), A);                // (p = 0 of a masked entry: 0 * finite)
      return p * w;
    }
    return p * A;
  };
  if (zero) {
    for (int i = v0 + tid; i < v1; i += GROUP) {
      if (i < nfull) hd_store16<T>(dx + (long long)i * VE, hd_u32x4{0, 0, 0, 0});
      else
        for (int j = 0; j < tail; ++j) dx[(long long)i * VE + j] = T::round(0.f);
    }
    return;                                            // uniform over the group
  }
  // distill: the teacher's entries of this segment, read while the row is on its way
  struct Teacher { int i; float q; };                  // i < 0: unused, or in another segment
  __shared__ Teacher sh_t[MODE == MODE_DISTILL ? 256 / GROUP : 1][MODE == MODE_DISTILL ? kTeacher : 1];
  const int own = GROUP == 256 ? 0 : threadIdx.x / GROUP, kept = a.k < kTeacher ? a.k : kTeacher;
  const float tm = MODE == MODE_DISTILL ? a.stats[4 * row + 2] : 0.f, tls2 = MODE == MODE_DISTILL ? a.stats[4 * row + 3] : 0.f;
  const long long e0 = (long long)v0 * VE, e1 = (long long)v1 * VE < a.V ? (long long)v1 * VE : a.V;
  auto entry = [&](int j) -> Teacher {
    const long long i = a.t_idx[row * a.k + j];
    if (i < e0 || i >= e1) return Teacher{-1, 0.f};
    return Teacher{(int)i, hd_exp2((lp_teacher(a, row * a.k + j) - tm) * c - tls2)};
  };
  if constexpr (MODE == MODE_DISTILL) {
    for (int j = tid; j < kept; j += GROUP) sh_t[own][j] = entry(j);
  }
  const int yv = y >= 0 ? (int)(y / VE) : -1, yj = y >= 0 ? (int)(y % VE) : 0;
  auto one = [&](int i, hd_u32x4 w) {
    float f[VE];
    T::unpack(w, f);
#pragma unroll
    for (int j = 0; j < VE; ++j) f[j] = grad(f[j]);
    if constexpr (MODE == MODE_LABEL) {
      if (i == yv) {
#pragma unroll
        for (int j = 0; j < VE; ++j) f[j] += j == yj ? g1 : 0.f;
      }
    }
    hd_store16<T>(dx + (long long)i * VE, T::pack(f));
  };
  if (v0 + GROUP * U <= nfull) {
    hd_u32x4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = hd_load16<T>(x + (long long)(v0 + u * GROUP + tid) * VE);
#pragma unroll
    for (int u = 0; u < U; ++u) one(v0 + u * GROUP + tid, w[u]);
  } else {
    for (int i = v0 + tid; i < v1; i += GROUP) {
      if (i < nfull) one(i, hd_load16<T>(x + (long long)i * VE));
      else
        for (int j = 0; j < tail; ++j) {
          float f = grad(T::load(x + (long long)i * VE + j));
          if (MODE == MODE_LABEL && i == yv && j == yj) f += g1;
          dx[(long long)i * VE + j] = T::round(f);
        }
    }
  }
  if constexpr (MODE == MODE_DISTILL) {
    // the teacher's entries of this segment again, whole: an index that occurs more than once takes the sum of its q.
    // (also after the stores above; one wave: program order)
    if constexpr (GROUP == 256) __syncthreads();
    else __builtin_amdgcn_wave_barrier();
    for (int j = tid; j < a.k; j += GROUP) {
      const Teacher me = j < kTeacher ? sh_t[own][j] : entry(j);
      if (me.i < 0) continue;
      float q = 0.f;
      int before = 0;
#pragma unroll 8
      for (int n = 0; n < kept; ++n) {
        const Teacher o = sh_t[own][n];
        q += o.i == me.i ? o.q : 0.f;
        before |= o.i == me.i && n < j ? 1 : 0;
      }
      for (int n = kept; n < a.k; ++n) {
        const Teacher o = entry(n);
        q += o.i == me.i ? o.q : 0.f;
        before |= o.i == me.i && n < j ? 1 : 0;
      }
      if (before) continue;
      const float p = hd_exp2(__fmaf_rn(T::load(x + me.i) - m, c, -ls2));
      dx[me.i] = T::round((p - q) * A);
    }
  }
}

// Segments of a row: where rows are few and long, the workgroup that owned one would be bound by its own arithmetic while most of the
// chip idles.  The second launch costs about 3 us, so a row has to pass what 1024 threads read in one round (16-bit) or two (fp32).
// One row, whole against segments, us a call (label statistics; with 20 alternatives; distillation):
//   bf16   65536  6.7 -  9.3, 10.9 - 10.8, 6.0 - 7.2     fp32   65536  6.7 - 8.1, 11.0 - 10.2, 6.3 - 7.6
//          65544 10.2 -  9.0, 15.0 - 11.3, 8.9 - 7.7            70000  8.5 - 8.3, 12.8 - 10.4, 7.8 - 7.9
//         100000 10.4 -  7.6, 15.8 - 11.2, 9.0 - 7.0           100000 10.2 - 8.0, 15.0 - 10.7, 9.0 - 7.5
//         131072 10.1 -  8.1, 15.0 - 10.9, 8.8 - 7.6           131072 10.1 - 8.1, 14.8 - 10.0, 8.9 - 7.7
// 64 rows of 131072: bf16 10.7 - 7.9, 15.6 - 14.3, 9.2 - 8.4, fp32 11.1 - 8.3, 15.9 - 15.0, 10.1 - 9.4; 128 rows fill half the chip by
// themselves (16.1 - 17.5 with alternatives).
struct Split {
  int nseg, seg;
  size_t keys, part;        // bytes
};
Split lp_split(long long T, int V, int dtype, int top) {
  const int ve = dtype == PN2_DT_F32 ? 4 : 8, nvec = V / ve + (V % ve != 0);
  if (T < 1 || T > 64 || V <= 65536) return Split{1, V, 0, 0};
  int n = nvec / 1024;
  if (n > kMaxSeg) n = kMaxSeg;
  const int each = (nvec + n - 1) / n;
  n = (nvec + each - 1) / each;
  return Split{n, each * ve, top ? (size_t)T * n * kSegThreads * 8 : 0, (size_t)T * n * 16};
}

template <class T, int MODE, bool TOP>
void lp_row_launch(const FwdArgs &a, hipStream_t st) {
  if (a.nseg > 1) {
    lp_row_kernel<T, MODE, TOP, kSegThreads, 4, true><<<(unsigned)(a.T * a.nseg), kSegThreads, 0, st>>>(a);
    lp_join_kernel<T, MODE, TOP, TOP ? 1024 : 256><<<(unsigned)a.T, TOP ? 1024 : 256, 0, st>>>(a);
    return;
  }
  // Fewer rows than CUs: one big workgroup per row with its loads on their way at once (1 x 131072 bf16 with 20 alternatives 15 us, 25
  // with 512 threads).  Otherwise several workgroups per CU, smaller ones for short rows, whose time is the selection's round trips
  // (8192 x 16384 bf16 with 20 alternatives: 95 us with 256 threads, 122 with 512; 8192 x 131072: 0.43 ms with 512).
  const int nvec = (a.V + T::kPerVec - 1) / T::kPerVec;
  if (nvec > 1024 && a.T <= 256) lp_row_kernel<T, MODE, TOP, 1024, 8, false><<<hd_grid(a.T, 1024), 1024, 0, st>>>(a);
  else if (nvec <= 4096) lp_row_kernel<T, MODE, TOP, 256, 4, false><<<hd_grid(a.T, 256), 256, 0, st>>>(a);
  else lp_row_kernel<T, MODE, TOP, 512, 4, false><<<hd_grid(a.T, 512), 512, 0, st>>>(a);
}

template <class T, int MODE>
int lp_forward(const FwdArgs &a, hipStream_t st) {
  if (a.V <= kSmallV) {
    const dim3 grid = hd_grid((a.T + 3) / 4, 256);
    if (a.V <= 64) lp_small_kernel<T, MODE, 1><<<grid, 256, 0, st>>>(a);
    else if (a.V <= 256) lp_small_kernel<T, MODE, 4><<<grid, 256, 0, st>>>(a);
    else if (a.V <= 1024) lp_small_kernel<T, MODE, 16><<<grid, 256, 0, st>>>(a);
    else lp_small_kernel<T, MODE, 32><<<grid, 256, 0, st>>>(a);
    return pn2_check_launch();
  }
  if constexpr (MODE == MODE_LABEL) {
    if (a.top) {
      lp_row_launch<T, MODE, true>(a, st);
      return pn2_check_launch();
    }
  }
  lp_row_launch<T, MODE, false>(a, st);
  return pn2_check_launch();
}

template <class T, int MODE>
int lp_backward(BwdArgs a, hipStream_t st) {
  constexpr int VE = T::kPerVec;
  const int nvec = (a.V + VE - 1) / VE;
  if (a.V <= kSmallV) {
    a.nseg = (nvec + 255) / 256;                       // 64 lanes x 4 vectors
    const long long units = a.T * a.nseg;
    lp_grad_kernel<T, MODE, 64><<<hd_grid((units + 3) / 4, 256), 256, 0, st>>>(a);
  } else {
    a.nseg = (nvec + 1023) / 1024;
    const long long units = a.T * a.nseg;
    lp_grad_kernel<T, MODE, 256><<<hd_grid(units, 256), 256, 0, st>>>(a);
  }
  return pn2_check_launch();
}

template <int MODE>
int lp_forward_any(int dtype, const FwdArgs &a, hipStream_t st) {
  if (dtype == PN2_DT_F32) return lp_forward<HdF32, MODE>(a, st);
  if (dtype == PN2_DT_BF16) return lp_forward<HdBF16, MODE>(a, st);
  return lp_forward<HdF16, MODE>(a, st);
}
template <int MODE>
int lp_backward_any(int dtype, const BwdArgs &a, hipStream_t st) {
  if (dtype == PN2_DT_F32) return lp_backward<HdF32, MODE>(a, st);
  if (dtype == PN2_DT_BF16) return lp_backward<HdBF16, MODE>(a, st);
  return lp_backward<HdF16, MODE>(a, st);
}

inline bool lp_bad(long long T, int V, long long ld, int dtype) {
  return T < 0 || V < 1 || ld < 0 || T > 0x7fffffffLL || dtype < PN2_DT_F32 || dtype > PN2_DT_F16;
}

// the caller's workspace divided
int lp_segments(FwdArgs &a, int dtype, void *workspace, size_t bytes) {
  const Split p = lp_split(a.T, a.V, dtype, a.top);
  if (bytes < p.keys + p.part) return PN2_ENOSPC;
  if (p.nseg > 1 && !workspace) return PN2_ENULL;
  a.nseg = p.nseg;
  a.seg = p.seg;
  a.keys = (u64 *)workspace;
  a.part = (float *)((char *)workspace + p.keys);
  return PN2_OK;
}

}  // namespace

extern "C" size_t pn2_label_logprobs_workspace_bytes(long long T, int V, int dtype, int top) {
  if (lp_bad(T, V, 0, dtype) || top < 0 || top > kMaxTop || top > V) return 0;
  const Split p = lp_split(T, V, dtype, top);
  return p.keys + p.part;
}

extern "C" size_t pn2_distill_topk_workspace_bytes(long long T, int V, int dtype) {
  if (lp_bad(T, V, 0, dtype)) return 0;
  return lp_split(T, V, dtype, 0).part;
}

extern "C" int pn2_label_logprobs(long long T, int V, long long ld, int dtype, const void *logits, const long long *labels,
                                  long long ignore_index, int top, float *log_prob, float *entropy, float *stats,
                                  float *top_log_prob, long long *top_index, void *workspace, size_t workspace_bytes, void *stream) {
  if (lp_bad(T, V, ld, dtype) || top < 0 || top > kMaxTop || top > V) return PN2_EINVAL;
  if (T == 0) return PN2_OK;
  if (!logits || !labels || !log_prob || !entropy || (top && (!top_log_prob || !top_index))) return PN2_ENULL;
  FwdArgs a{};
  a.T = T; a.ld = ld; a.V = V; a.top = top; a.c = kHdLog2e; a.tau = 1.f;
  a.logits = logits; a.labels = labels; a.ignore = ignore_index;
  a.log_prob = log_prob; a.entropy = entropy; a.stats = stats; a.top_lp = top_log_prob; a.top_idx = top_index;
  const int rc = lp_segments(a, dtype, workspace, workspace_bytes);
  if (rc != PN2_OK) return rc;
  return lp_forward_any<MODE_LABEL>(dtype, a, (hipStream_t)stream);
}

extern "C" int pn2_label_logprobs_grad(long long T, int V, long long ld, int dtype, const void *logits, const long long *labels,
                                       long long ignore_index, const float *stats, const float *entropy, const float *g_log_prob,
                                       const float *g_entropy, void *dlogits, void *stream) {
  if (lp_bad(T, V, ld, dtype)) return PN2_EINVAL;
  if (T == 0) return PN2_OK;
  if (!logits || !labels || !stats || !entropy || !dlogits) return PN2_ENULL;
  BwdArgs a{};
  a.T = T; a.ld = ld; a.V = V; a.c = kHdLog2e; a.tau = 1.f;
  a.logits = logits; a.labels = labels; a.ignore = ignore_index;
  a.stats = stats; a.entropy = entropy; a.g_lp = g_log_prob; a.g_ent = g_entropy; a.dlogits = dlogits;
  return lp_backward_any<MODE_LABEL>(dtype, a, (hipStream_t)stream);
}

extern "C" int pn2_distill_topk(long long T, int V, long long ld, int dtype, const void *logits, int k, const long long *teacher_index,
                                int teacher_dtype, const void *teacher_logits, float temperature, float *loss, float *stats,
                                void *workspace, size_t workspace_bytes, void *stream) {
  if (lp_bad(T, V, ld, dtype) || k < 1 || teacher_dtype < PN2_DT_F32 || teacher_dtype > PN2_DT_F16 || !(temperature > 0.f) ||
      !(temperature < kHdInf))
    return PN2_EINVAL;
  if (T == 0) return PN2_OK;
  if (!logits || !teacher_index || !teacher_logits || !loss) return PN2_ENULL;
  FwdArgs a{};
  a.T = T; a.ld = ld; a.V = V; a.k = k; a.tau = temperature; a.c = kHdLog2e / temperature;
  a.logits = logits; a.t_idx = teacher_index; a.t_val = teacher_logits; a.t_dtype = teacher_dtype; a.loss = loss; a.stats = stats;
  const int rc = lp_segments(a, dtype, workspace, workspace_bytes);
  if (rc != PN2_OK) return rc;
  return lp_forward_any<MODE_DISTILL>(dtype, a, (hipStream_t)stream);
}

extern "C" int pn2_distill_topk_grad(long long T, int V, long long ld, int dtype, const void *logits, int k,
                                     const long long *teacher_index, int teacher_dtype, const void *teacher_logits,
                                     float temperature, const float *stats, const float *g_loss, void *dlogits, void *stream) {
  if (lp_bad(T, V, ld, dtype) || k < 1 || teacher_dtype < PN2_DT_F32 || teacher_dtype > PN2_DT_F16 || !(temperature > 0.f) ||
      !(temperature < kHdInf))
    return PN2_EINVAL;
  if (T == 0) return PN2_OK;
  if (!logits || !teacher_index || !teacher_logits || !stats || !g_loss || !dlogits) return PN2_ENULL;
  BwdArgs a{};
  a.T = T; a.ld = ld; a.V = V; a.k = k; a.tau = temperature; a.c = kHdLog2e / temperature;
  a.logits = logits; a.t_idx = teacher_index; a.t_val = teacher_logits; a.t_dtype = teacher_dtype;
  a.stats = stats; a.g_loss = g_loss; a.dlogits = dlogits;
  return lp_backward_any<MODE_DISTILL>(dtype, a, (hipStream_t)stream);
}
