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
// of the row; the k best elements of a row lie in the shares of the k threads with the best keys (an element of another
// thread has k better keys above it), so only those shares are looked at again (from L2): k / BT of the row.
#include "head_common.h"

namespace {

constexpr int kMaxTop = 64;              // one list entry per lane
constexpr int kSmallV = 1024;            // up to here: one wave per row, the row in registers

// order-preserving map float -> unsigned (-0 = +0; -inf -> kKeyNegInf; 0 = "nothing")
constexpr unsigned kKeyNegInf = 0x007fffffu;
__device__ __forceinline__ unsigned lp_key(float v) {
  const unsigned b = __builtin_bit_cast(unsigned, v + 0.f);
  return (int)b < 0 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float lp_unkey(unsigned k) {
  return __builtin_bit_cast(float, (int)k < 0 ? k & 0x7fffffffu : ~k);
}

// lane i <- lane i - 1 (lane 0 keeps its own)
__device__ __forceinline__ unsigned lp_shift_up(unsigned v) {
  return (unsigned)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x138, 0xF, 0xF, false);   // wave_shr:1
}

// A descending list of 64 (key, index) pairs, one per lane; equal keys in ascending index order; key 0 = empty.
struct TopList {
  unsigned key;
  int idx;
  __device__ __forceinline__ void clear() { key = 0u; idx = 0x7fffffff; }
  __device__ __forceinline__ bool above(unsigned k, int i) const { return key > k || (key == k && idx < i); }
  __device__ __forceinline__ void insert(unsigned k, int i) {          // (k, i) wave-uniform
    const int pos = __popcll(__ballot(above(k, i)));
    const int lane = pn2_lane();
    const unsigned pk = lp_shift_up(key);
    const int pi = (int)lp_shift_up((unsigned)idx);
    key = lane > pos ? pk : (lane == pos ? k : key);
    idx = lane > pos ? pi : (lane == pos ? i : idx);
  }
};

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
};

__device__ __forceinline__ float lp_teacher(const FwdArgs &a, long long at) {
  if (a.t_dtype == PN2_DT_F32) return ((const float *)a.t_val)[at];
  if (a.t_dtype == PN2_DT_BF16) return (float)((const __bf16 *)a.t_val)[at];
  return (float)((const _Float16 *)a.t_val)[at];
}

// One wave finishes a label row: stats are wave-uniform.
template <class T>
__device__ __forceinline__ void lp_finish_label(const FwdArgs &a, long long row, const typename T::elem *x, const RowStat &r) {
  if (pn2_lane() == 0) {
    const long long y = a.labels[row];
    float lp = 0.f;
    if (y != a.ignore) {
      if (y < 0 || y >= a.V) lp = __builtin_nanf("");
      else lp = lp_logp(T::load(x + y), r);
    }
    a.log_prob[row] = lp;
    a.entropy[row] = r.entropy;
    if (a.stats) {
      a.stats[2 * row] = r.m;
      a.stats[2 * row + 1] = r.ls2;
    }
  }
}

// One wave finishes a distillation row.  An unused slot has a negative index or the value -inf; a row without a used slot
// has no loss (and its logits were not read: r is not looked at).  An index >= V makes the row NaN.
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
    if (i >= 0) tm = fmaxf(tm, lp_teacher(a, at + j));
    bad |= i >= a.V;
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

__device__ __forceinline__ void lp_write_top(const FwdArgs &a, long long row, const TopList &l, const RowStat &r) {
  const int lane = pn2_lane();
  if (lane >= a.top) return;
  const bool none = l.key <= kKeyNegInf || r.nan;
  a.top_lp[row * a.top + lane] = r.nan ? __builtin_nanf("") : (none ? -kHdInf : lp_logp(lp_unkey(l.key), r));
  a.top_idx[row * a.top + lane] = none ? -1 : l.idx;
}

enum { MODE_LABEL, MODE_DISTILL };

// ------------------------------------------------------------------------------------------------ V <= 1024: a wave per row
template <class T, int MODE, int EPL>
__global__ __launch_bounds__(256) void lp_small_kernel(FwdArgs a) {
  const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
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
  float v[EPL];
  float m = -kHdInf;
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    const int i = lane + j * PN2_WAVE;
    v[j] = i < a.V ? T::load(x + i) : -kHdInf;
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
    lp_finish_label<T>(a, row, x, f);
    if (a.top) {
      TopList l;
      l.clear();
      for (int q = 0; q < a.top; ++q) {
        unsigned bk = 0u, bi = 0u;
#pragma unroll
        for (int j = 0; j < EPL; ++j) {
          const unsigned k = lp_key(v[j]);
          const bool better = k > bk;
          bk = better ? k : bk;
          bi = better ? ~(unsigned)(lane + j * PN2_WAVE) : bi;
        }
        unsigned mk, mi;
        pn2_wave_argmax_u32x2(bk, bi, mk, mi);
        if (mk <= kKeyNegInf) break;
        const int at = (int)~mi;
        if (lane == q) { l.key = mk; l.idx = at; }
#pragma unroll
        for (int j = 0; j < EPL; ++j)
          if (at == lane + j * PN2_WAVE) v[j] = -kHdInf;
      }
      lp_write_top(a, row, l, f);
    }
  }
}

// --------------------------------------------------------------------------------------------- V > 1024: a workgroup per row
template <class T, int MODE, bool TOP, int BT>
__global__ __launch_bounds__(BT) void lp_row_kernel(FwdArgs a) {
  constexpr int VE = T::kPerVec, U = 4, W = BT / PN2_WAVE;
  constexpr bool ENT = MODE == MODE_LABEL;
  typedef typename T::elem elem;
  __shared__ float sh_m[W], sh_s[W], sh_se[W];
  const long long row = blockIdx.x;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const elem *x = (const elem *)a.logits + row * a.ld;
  RowSum r{-kHdInf, 0.f, 0.f, 0.f};
  if constexpr (MODE == MODE_DISTILL) {
    if (!lp_teacher_any(a, row)) {                     // the same answer in every wave
      if (wave == 0) lp_finish_distill<T>(a, row, x, RowStat{}, false);
      return;
    }
  }
  const float c = a.c, lim = lp_lim(c);
  r.M2 = lp_ref(r.m, c, lim);
  const int nfull = a.V / VE, tail = a.V % VE;
  int ord = 0x7fffffff;                                // first vector that holds the thread's maximum
  int b = 0;
  for (; b + BT * U <= nfull; b += BT * U) {
    hd_u32x4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = hd_load16<T>(x + (long long)(b + u * BT + tid) * VE);
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
  for (int i = b + tid; i < nfull + (tail != 0); i += BT) {
    float g[VE];
    if (i < nfull) {
      T::unpack(hd_load16<T>(x + (long long)i * VE), g);
    } else {
#pragma unroll
      for (int j = 0; j < VE; ++j) g[j] = j < tail ? T::load(x + (long long)i * VE + j) : -kHdInf;
    }
    float vm = g[0];
#pragma unroll
    for (int j = 1; j < VE; ++j) vm = fmaxf(vm, g[j]);
    if constexpr (TOP) {
      if (vm > r.m) ord = i;
    }
    lp_add<ENT>(r, g, vm, c, lim);
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
  float res = __fmaf_rn(r.m, c, -r.M2);
  if (fabsf(r.m) > lim && fabsf(r.m) < kHdInf) {
    // x c may overflow: sum again with (x - m) c.  Uniform over the workgroup; every wave has passed the barrier above.
    float s = 0.f, se = 0.f;
    for (int i = tid; i < a.V; i += BT) {
      const float t = (T::load(x + i) - r.m) * c, e = hd_exp2(t);
      s += e;
      if constexpr (ENT) se += e * fmaxf(t, -1e30f);
    }
    s = hd_wave_sum(s);
    se = hd_wave_sum(se);
    __syncthreads();
    if (lane == 0) { sh_s[wave] = s; sh_se[wave] = se; }
    __syncthreads();
    r.s = r.se = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) { r.s += sh_s[w]; r.se += sh_se[w]; }
    res = 0.f;
  }
  const RowStat st = lp_stat(r, res);
  if constexpr (MODE == MODE_DISTILL) {
    if (wave == 0) lp_finish_distill<T>(a, row, x, st, true);
    return;
  }
  if (wave == W - 1) lp_finish_label<T>(a, row, x, st);
  if constexpr (TOP) {
    __shared__ unsigned sh_key[BT];
    __shared__ int sh_ord[BT];
    __shared__ int sh_win[kMaxTop];
    __shared__ int sh_nwin;
    __shared__ unsigned sh_lkey[W][kMaxTop];
    __shared__ int sh_lidx[W][kMaxTop];
    const unsigned okey = own == -kHdInf ? 0u : lp_key(own);
    sh_key[tid] = okey;
    sh_ord[tid] = ord;
    __syncthreads();
    if (wave == 0) {
      // the `top` best of the threads' keys: W keys per lane, one wave-wide arg-max per winner
      constexpr int R = W;
      unsigned key[R], inv[R];
#pragma unroll
      for (int q = 0; q < R; ++q) {
        key[q] = sh_key[q * PN2_WAVE + lane];
        inv[q] = ~(unsigned)sh_ord[q * PN2_WAVE + lane];
      }
      int n = 0;
      for (; n < a.top; ++n) {
        unsigned bk = 0u, bi = 0u;
        int bq = 0;
#pragma unroll
        for (int q = 0; q < R; ++q) {
          const bool better = key[q] > bk || (key[q] == bk && inv[q] > bi);
          bk = better ? key[q] : bk;
          bi = better ? inv[q] : bi;
          bq = better ? q : bq;
        }
        unsigned mk, mi;
        const u64 who = pn2_wave_argmax_u32x2(bk, bi, mk, mi);
        if (mk == 0u) break;
        if (lane == __ffsll((unsigned long long)who) - 1) {
          sh_win[n] = bq * PN2_WAVE + lane;
#pragma unroll
          for (int q = 0; q < R; ++q)
            if (q == bq) key[q] = 0u;
        }
      }
      if (lane == 0) sh_nwin = n;
    }
    __syncthreads();
    const int nwin = sh_nwin;
    // the k-th key bounds the elements from below (fewer winners than `top`: everything counts)
    const int last = nwin == a.top ? sh_win[nwin - 1] : -1;
    const unsigned low_key = last >= 0 ? sh_key[last] : kKeyNegInf + 1;
    const int low_ord = last >= 0 ? sh_ord[last] : 0x7fffffff;
    TopList l;
    l.clear();
    const int nvec = nfull + (tail != 0);
    for (int w = wave; w < nwin; w += W) {
      const int t = sh_win[w];
      for (int s0 = t; s0 < nvec; s0 += BT * PN2_WAVE) {           // the share of thread t, a vector per lane
        const int i = s0 + lane * BT;
        float g[VE];
        if (i < nfull) {
          T::unpack(hd_load16<T>(x + (long long)i * VE), g);
        } else {
#pragma unroll
          for (int j = 0; j < VE; ++j) g[j] = i == nfull && j < tail ? T::load(x + (long long)i * VE + j) : -kHdInf;
        }
#pragma unroll
        for (int j = 0; j < VE; ++j) {
          const unsigned k = lp_key(g[j]);
          bool cand = k > low_key || (k == low_key && i <= low_ord);
          cand = cand && i < nvec && k > kKeyNegInf && g[j] == g[j];
          u64 todo = __ballot(cand);
          while (todo) {
            const int src = __ffsll((unsigned long long)todo) - 1;
            todo &= todo - 1;
            l.insert((unsigned)__builtin_amdgcn_readlane((int)k, src), __builtin_amdgcn_readlane(i, src) * VE + j);
          }
        }
      }
    }
    sh_lkey[wave][lane] = l.key;
    sh_lidx[wave][lane] = l.idx;
    __syncthreads();
    if (wave == 0) {
      for (int w = 1; w < W; ++w) {
        const unsigned k = sh_lkey[w][lane];
        const int i = sh_lidx[w][lane];
        // (a list is sorted: its used entries are the first ones)
        u64 todo = __ballot(k != 0u);
        while (todo) {
          const int src = __ffsll((unsigned long long)todo) - 1;
          todo &= todo - 1;
          l.insert((unsigned)__builtin_amdgcn_readlane((int)k, src), __builtin_amdgcn_readlane(i, src));
        }
      }
      lp_write_top(a, row, l, st);
    }
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

// GROUP threads own a segment of one row.  Bound by its bytes (V read, V written); ~6 vector instructions per element.
template <class T, int MODE, int GROUP>
__global__ __launch_bounds__(256) void lp_grad_kernel(BwdArgs a) {
  constexpr int VE = T::kPerVec, U = 4;
  typedef typename T::elem elem;
  const int tid = threadIdx.x % GROUP;
  const long long unit = GROUP == 256 ? (long long)blockIdx.x : (long long)blockIdx.x * (256 / GROUP) + threadIdx.x / GROUP;
  const long long row = unit / a.nseg;
  if (row >= a.T) return;                              // (GROUP < 256 only: no barrier below is left behind)
  const int seg = (int)(unit - row * a.nseg);
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
    // the teacher's entries of this segment again, whole: an index that occurs more than once takes the sum of its q
    if constexpr (GROUP == 256) __syncthreads();       // after the stores above (one wave: program order)
    const float tm = a.stats[4 * row + 2], tls2 = a.stats[4 * row + 3];
    const long long at = row * a.k, e0 = (long long)v0 * VE, e1 = (long long)v1 * VE < a.V ? (long long)v1 * VE : a.V;
    for (int j = tid; j < a.k; j += GROUP) {
      const long long i = a.t_idx[at + j];
      if (i < e0 || i >= e1) continue;
      bool first = true;
      for (int n = 0; n < j && first; ++n) first = a.t_idx[at + n] != i;
      if (!first) continue;
      float q = 0.f;
      for (int n = j; n < a.k; ++n)
        if (a.t_idx[at + n] == i) q += hd_exp2((lp_teacher(a, at + n) - tm) * c - tls2);
      const float p = hd_exp2(__fmaf_rn(T::load(x + i) - m, c, -ls2));
      dx[i] = T::round((p - q) * A);
    }
  }
}

template <class T, int MODE>
int lp_forward(const FwdArgs &a, hipStream_t st) {
  if (a.V <= kSmallV) {
    const unsigned grid = (unsigned)((a.T + 3) / 4);
    if (a.V <= 64) lp_small_kernel<T, MODE, 1><<<grid, 256, 0, st>>>(a);
    else if (a.V <= 256) lp_small_kernel<T, MODE, 4><<<grid, 256, 0, st>>>(a);
    else lp_small_kernel<T, MODE, 16><<<grid, 256, 0, st>>>(a);
    return pn2_check_launch();
  }
  const unsigned grid = (unsigned)a.T;
  if (MODE == MODE_LABEL && a.top) lp_row_kernel<T, MODE, true, 512><<<grid, 512, 0, st>>>(a);
  else lp_row_kernel<T, MODE, false, 512><<<grid, 512, 0, st>>>(a);
  return pn2_check_launch();
}

template <class T, int MODE>
int lp_backward(BwdArgs a, hipStream_t st) {
  constexpr int VE = T::kPerVec;
  const int nvec = (a.V + VE - 1) / VE;
  if (a.V <= kSmallV) {
    a.nseg = (nvec + 255) / 256;                       // 64 lanes x 4 vectors
    const long long units = a.T * a.nseg;
    lp_grad_kernel<T, MODE, 64><<<(unsigned)((units + 3) / 4), 256, 0, st>>>(a);
  } else {
    a.nseg = (nvec + 1023) / 1024;
    const long long units = a.T * a.nseg;
    if (units > 0x7fffffffLL) return PN2_EINVAL;
    lp_grad_kernel<T, MODE, 256><<<(unsigned)units, 256, 0, st>>>(a);
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

}  // namespace

extern "C" int pn2_label_logprobs(long long T, int V, long long ld, int dtype, const void *logits, const long long *labels,
                                  long long ignore_index, int top, float *log_prob, float *entropy, float *stats,
                                  float *top_log_prob, long long *top_index, void *stream) {
  if (lp_bad(T, V, ld, dtype) || top < 0 || top > kMaxTop || top > V) return PN2_EINVAL;
  if (T == 0) return PN2_OK;
  if (!logits || !labels || !log_prob || !entropy || (top && (!top_log_prob || !top_index))) return PN2_ENULL;
  FwdArgs a{};
  a.T = T; a.ld = ld; a.V = V; a.top = top; a.c = kHdLog2e; a.tau = 1.f;
  a.logits = logits; a.labels = labels; a.ignore = ignore_index;
  a.log_prob = log_prob; a.entropy = entropy; a.stats = stats; a.top_lp = top_log_prob; a.top_idx = top_index;
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
                                void *stream) {
  if (lp_bad(T, V, ld, dtype) || k < 1 || teacher_dtype < PN2_DT_F32 || teacher_dtype > PN2_DT_F16 || !(temperature > 0.f) ||
      !(temperature < kHdInf))
    return PN2_EINVAL;
  if (T == 0) return PN2_OK;
  if (!logits || !teacher_index || !teacher_logits || !loss) return PN2_ENULL;
  FwdArgs a{};
  a.T = T; a.ld = ld; a.V = V; a.k = k; a.tau = temperature; a.c = kHdLog2e / temperature;
  a.logits = logits; a.t_idx = teacher_index; a.t_val = teacher_logits; a.t_dtype = teacher_dtype; a.loss = loss; a.stats = stats;
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
