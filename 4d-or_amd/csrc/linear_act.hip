// linear_act.hip — y = act(x W^T + b) + r with its backward pass: the dense layer of the heads, any M, N, K, fp32 / bf16 / fp16.
//
//   forward    z = x W^T + b,  y = act(z) + r,  slope d = act'(z) kept for the backward pass
//   backward   dz = dy d,  dx = dz W,  dW = dz^T x,  db = sum over rows of dz
//
// All three products are  C[i][j] = sum_k P(i, k) Q(j, k)  with P, Q contiguous either along k ("K" operands: x and W of the
// forward product, dz of dx) or along their row ("R" operands: W of dx, dz and x of dW).  Products accumulate in fp32 on the
// matrix cores (v_mfma_f32_16x16x32 for 16-bit types, v_mfma_f32_16x16x4_f32 for fp32); bias, activation, slope and residual are
// fp32 in the epilogue; each output is rounded once.  The SLOPE is what is stored, not z: rounding d costs every dz a relative
// half-step, rounding z would cost an absolute one where d crosses zero.  Slopes lie in [-0.2, 1.2], so 16-bit types store them
// as fp16 (2^-11; bf16 would be 2^-8 for the same bytes); dz is rounded to the operands' type for the matrix cores.
//
// The matrix instruction takes Q as its row operand and P as its column operand, so a lane of the result holds one row i of C
// and four consecutive columns j: bias, residual and stores are contiguous per lane.
#include "head_common.h"

namespace {

typedef float la_f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 la_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 la_f16x8 __attribute__((ext_vector_type(8)));

enum { ACT_NONE, ACT_RELU, ACT_GELU, ACT_GELU_TANH, ACT_SILU };

// 16-byte fragments: 8 16-bit contraction indices per lane, or 4 fp32 ones (lane group g of 16 holds k = 4 g .. 4 g + 3; the
// four instructions take k = {i, 4 + i, 8 + i, 12 + i}: any order is right as long as both operands use it)
__device__ __forceinline__ la_f32x4 la_mma(HdBF16, hd_u32x4 q, hd_u32x4 p, la_f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(la_bf16x8, q), __builtin_bit_cast(la_bf16x8, p), c, 0, 0, 0);
}
__device__ __forceinline__ la_f32x4 la_mma(HdF16, hd_u32x4 q, hd_u32x4 p, la_f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(la_f16x8, q), __builtin_bit_cast(la_f16x8, p), c, 0, 0, 0);
}
__device__ __forceinline__ la_f32x4 la_mma(HdF32, hd_u32x4 q, hd_u32x4 p, la_f32x4 c) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned qi = q[i], pi = p[i];
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, qi), __builtin_bit_cast(float, pi), c, 0, 0, 0);
  }
  return c;
}

// act(z) and its slope
template <int ACT>
__device__ __forceinline__ void la_act(float z, float &y, float &d) {
  if constexpr (ACT == ACT_NONE) {
    y = z;
    d = 1.f;
  } else if constexpr (ACT == ACT_RELU) {
    y = z <= 0.f ? 0.f : z;                            // (NaN stays NaN)
    d = z <= 0.f ? 0.f : 1.f;
  } else if constexpr (ACT == ACT_SILU) {
    const float s = __builtin_amdgcn_rcpf(1.f + hd_exp2(-kHdLog2e * z));
    y = z * s;
    d = __fmaf_rn(y, 1.f - s, s);
  } else if constexpr (ACT == ACT_GELU) {
    const float cdf = 0.5f + 0.5f * erff(z * 0.7071067811865476f);
    y = z * cdf;
    d = __fmaf_rn(z * 0.3989422804014327f, hd_exp2(-0.5f * kHdLog2e * z * z), cdf);
  } else {
    // (1 + tanh u) / 2 = 1 / (1 + e^(-2u)), u = sqrt(2/pi) (z + 0.044715 z^3); beyond |z| = 30 the gate is 0 or 1
    const float w = fminf(fmaxf(z, -30.f), 30.f), w2 = w * w;
    const float u2 = 1.5957691216057308f * w * __fmaf_rn(0.044715f, w2, 1.f);
    const float g = __builtin_amdgcn_rcpf(1.f + hd_exp2(-kHdLog2e * u2));
    y = z * g;
    d = __fmaf_rn(w * g * (1.f - g), 1.5957691216057308f * __fmaf_rn(0.134145f, w2, 1.f), g);
  }
}

struct Epilogue {
  const void *bias;         // (N) of bias_f32 ? float : the element type, or NULL
  int bias_f32;
  int act;
  const void *res;          // (M, N) at stride ldr, or NULL
  long long ldr;
  void *y;                  // (M, N) dense
  void *slope;              // (M, N) dense, fp32 for fp32 and fp16 for 16-bit types, or NULL
};

template <class T> struct SlopeOf { typedef HdF16 type; };
template <> struct SlopeOf<HdF32> { typedef HdF32 type; };

struct Product {
  long long M, N, K;
  const void *p, *q;
  long long ldp, ldq;
  int vecp, vecq;           // rows 16-byte aligned: vector loads
  int splits;
  long long kchunk;         // contraction indices per split (a multiple of the tile's)
  float *partial;           // splits > 1: (splits, M, N)
  Epilogue e;
};

template <class T>
__device__ __forceinline__ float la_bias(const Epilogue &e, long long j) {
  if (!e.bias) return 0.f;
  return e.bias_f32 ? ((const float *)e.bias)[j] : T::load((const typename T::elem *)e.bias + j);
}

template <class T>
__device__ __forceinline__ void la_finish_any(const Epilogue &e, long long N, long long i, long long j, float z) {
  typedef typename T::elem elem;
  z += la_bias<T>(e, j);
  float y, d;
  switch (e.act) {
    case ACT_RELU: la_act<ACT_RELU>(z, y, d); break;
    case ACT_GELU: la_act<ACT_GELU>(z, y, d); break;
    case ACT_GELU_TANH: la_act<ACT_GELU_TANH>(z, y, d); break;
    case ACT_SILU: la_act<ACT_SILU>(z, y, d); break;
    default: la_act<ACT_NONE>(z, y, d);
  }
  if (e.res) y += T::load((const elem *)e.res + i * e.ldr + j);
  ((elem *)e.y)[i * N + j] = T::round(y);
  typedef typename SlopeOf<T>::type S;
  if (e.slope) ((typename S::elem *)e.slope)[i * N + j] = S::round(d);
}

// A tile of 64 rows x 64 bytes of contraction (KB = 16 or 32 indices) goes through registers into LDS rows of 64 + 16 bytes.
// K operand: thread -> (row tid / 4, 16-byte piece tid % 4).  R operand: thread -> (index tid / (64 / VE), piece), stored
// transposed.  Rows and indices out of range are zero.
template <class T, bool ROWS>
struct TileLoad {
  typedef typename T::elem elem;
  static constexpr int VE = T::kPerVec, KB = 4 * VE, LDT = 80 / (int)sizeof(elem);
  hd_u32x4 w;
  __device__ __forceinline__ void fetch(const elem *g, long long ld, int vec, long long r0, long long R, long long k0, long long k1,
                                        int tid) {
    long long r, k, n;
    const elem *src;
    if constexpr (!ROWS) {
      r = r0 + tid / 4;
      k = k0 + (tid % 4) * VE;
      n = r < R ? k1 - k : 0;
      src = g + r * ld + k;
    } else {
      constexpr int PR = 64 / VE;
      k = k0 + tid / PR;
      r = r0 + (tid % PR) * VE;
      n = k < k1 ? R - r : 0;
      src = g + k * ld + r;
    }
    if (vec && n >= VE) {
      w = hd_load16<T>(src);
    } else {
      elem v[VE];
#pragma unroll
      for (int i = 0; i < VE; ++i) v[i] = i < n ? src[i] : T::round(0.f);
      __builtin_memcpy(&w, v, 16);
    }
  }
  __device__ __forceinline__ void store(elem *lds, int tid) const {
    if constexpr (!ROWS) {
      __builtin_memcpy((elem *)__builtin_assume_aligned(lds + (tid / 4) * LDT + (tid % 4) * VE, 16), &w, 16);
    } else {
      constexpr int PR = 64 / VE;
      elem v[VE];
      __builtin_memcpy(v, &w, 16);
#pragma unroll
      for (int i = 0; i < VE; ++i) lds[((tid % PR) * VE + i) * LDT + tid / PR] = v[i];
    }
  }
};

// 64 x 64 tile, four waves of 32 x 32, any alignment and any size.
template <class T, bool PROWS, bool QROWS>
__global__ __launch_bounds__(256) void la_any_kernel(Product a) {
  typedef typename T::elem elem;
  constexpr int KB = 4 * T::kPerVec, LDT = 80 / (int)sizeof(elem);
  __shared__ __align__(16) elem sp[64 * LDT], sq[64 * LDT];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const long long i0 = (long long)blockIdx.x * 64, j0 = (long long)blockIdx.y * 64;
  const long long k0 = (long long)blockIdx.z * a.kchunk, k1 = k0 + a.kchunk < a.K ? k0 + a.kchunk : a.K;
  const int wi = (wave & 1) * 32, wj = (wave >> 1) * 32;
  la_f32x4 acc[2][2] = {};
  TileLoad<T, PROWS> lp;
  TileLoad<T, QROWS> lq;
  lp.fetch((const elem *)a.p, a.ldp, a.vecp, i0, a.M, k0, k1, tid);
  lq.fetch((const elem *)a.q, a.ldq, a.vecq, j0, a.N, k0, k1, tid);
  for (long long k = k0; k < k1; k += KB) {
    lp.store(sp, tid);
    lq.store(sq, tid);
    __syncthreads();
    if (k + KB < k1) {
      lp.fetch((const elem *)a.p, a.ldp, a.vecp, i0, a.M, k + KB, k1, tid);
      lq.fetch((const elem *)a.q, a.ldq, a.vecq, j0, a.N, k + KB, k1, tid);
    }
    hd_u32x4 fp[2], fq[2];
    const int r = lane & 15, c = (lane >> 4) * T::kPerVec;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      __builtin_memcpy(&fp[t], __builtin_assume_aligned(sp + (wi + t * 16 + r) * LDT + c, 16), 16);
      __builtin_memcpy(&fq[t], __builtin_assume_aligned(sq + (wj + t * 16 + r) * LDT + c, 16), 16);
    }
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int u = 0; u < 2; ++u) acc[t][u] = la_mma(T{}, fq[u], fp[t], acc[t][u]);
    __syncthreads();
  }
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const long long i = i0 + wi + t * 16 + (lane & 15), j = j0 + wj + u * 16 + (lane >> 4) * 4 + n;
        if (i >= a.M || j >= a.N) continue;
        if (a.splits > 1) a.partial[((long long)blockIdx.z * a.M + i) * a.N + j] = acc[t][u][n];
        else la_finish_any<T>(a.e, a.N, i, j, acc[t][u][n]);
      }
}

// the split contraction joined in a fixed order, then the epilogue
template <class T>
__global__ __launch_bounds__(256) void la_join_kernel(Product a) {
  const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
  if (at >= a.M * a.N) return;
  float z = 0.f;
  for (int s = 0; s < a.splits; ++s) z += a.partial[(long long)s * a.M * a.N + at];
  la_finish_any<T>(a.e, a.N, at / a.N, at % a.N, z);
}

// dz = dy slope (dz NULL: only the sums) and the column sums of a strip of rows -> part (strips, N) fp32
template <class T>
__global__ __launch_bounds__(256) void la_dz_kernel(long long M, long long N, long long strip, const void *dy_, long long ldy,
                                                    const void *slope_, void *dz_, float *part) {
  typedef typename T::elem elem;
  typedef typename SlopeOf<T>::type S;
  const elem *dy = (const elem *)dy_;
  const typename S::elem *slope = (const typename S::elem *)slope_;
  elem *dz = (elem *)dz_;
  const long long j = (long long)blockIdx.x * 256 + threadIdx.x;
  if (j >= N) return;
  const long long i0 = (long long)blockIdx.y * strip, i1 = i0 + strip < M ? i0 + strip : M;
  float s = 0.f;
  for (long long i = i0; i < i1; ++i) {
    float v = T::load(dy + i * ldy + j);
    if (slope) v *= S::load(slope + i * N + j);
    if (dz) dz[i * N + j] = T::round(v);
    s += v;
  }
  if (part) part[(long long)blockIdx.y * N + j] = s;
}

template <class T>
__global__ __launch_bounds__(256) void la_db_kernel(long long N, long long strips, const float *part, void *db, int db_f32) {
  const long long j = (long long)blockIdx.x * 256 + threadIdx.x;
  if (j >= N) return;
  float s = 0.f;
  for (long long i = 0; i < strips; ++i) s += part[i * N + j];
  if (db_f32) ((float *)db)[j] = s;
  else ((typename T::elem *)db)[j] = T::round(s);
}

constexpr long long kMaxDim = 1LL << 31;

inline long long la_div(long long a, long long b) { return (a + b - 1) / b; }
inline size_t la_align(size_t n) { return (n + 255) & ~(size_t)255; }

// how often the contraction of a product is split: until two workgroups per CU run, at least four tiles of it each
void la_plan(Product &a, int dtype) {
  const long long kb = dtype == PN2_DT_F32 ? 16 : 32, tiles = la_div(a.M, 64) * la_div(a.N, 64), steps = la_div(a.K, kb);
  long long s = 512 / tiles;
  if (s > steps / 4) s = steps / 4;
  if (s < 1) s = 1;
  if (s > 64) s = 64;
  const long long per = la_div(steps, s);
  a.splits = (int)la_div(steps, per);
  a.kchunk = per * kb;
}

size_t la_product_bytes(long long M, long long N, long long K, int dtype) {
  Product a{};
  a.M = M; a.N = N; a.K = K;
  la_plan(a, dtype);
  return a.splits > 1 ? la_align((size_t)a.splits * M * N * 4) : 0;
}

bool la_vec(const void *p, long long ld, int dtype) {
  const long long es = dtype == PN2_DT_F32 ? 4 : 2;
  return ((uintptr_t)p & 15) == 0 && (ld * es) % 16 == 0;
}

template <class T, bool PROWS, bool QROWS>
int la_product(Product a, int dtype, void *ws, size_t ws_bytes, hipStream_t st) {
  la_plan(a, dtype);
  const size_t need = a.splits > 1 ? la_align((size_t)a.splits * a.M * a.N * 4) : 0;
  if (ws_bytes < need) return PN2_ENOSPC;
  if (need && !ws) return PN2_ENULL;
  a.partial = (float *)ws;
  a.vecp = la_vec(a.p, a.ldp, dtype);
  a.vecq = la_vec(a.q, a.ldq, dtype);
  const long long gx = la_div(a.M, 64), gy = la_div(a.N, 64);
  if (gy > 65535) return PN2_EINVAL;
  la_any_kernel<T, PROWS, QROWS><<<dim3((unsigned)gx, (unsigned)gy, (unsigned)a.splits), 256, 0, st>>>(a);
  if (a.splits > 1) la_join_kernel<T><<<(unsigned)la_div(a.M * a.N, 256), 256, 0, st>>>(a);
  return pn2_check_launch();
}

inline bool la_bad(long long M, long long N, long long K, int dtype) {
  return M < 0 || N < 1 || K < 1 || M >= kMaxDim || N > 65535LL * 64 || K > 65535LL * 64 || dtype < PN2_DT_F32 || dtype > PN2_DT_F16;
}

constexpr long long kStripRows = 64;          // rows per partial column sum (at most 1024 strips)
inline long long la_strip(long long M) {
  const long long s = la_div(M, 1024);
  return s > kStripRows ? s : kStripRows;
}

template <class T>
int la_forward(Product a, int dtype, void *ws, size_t ws_bytes, hipStream_t st) {
  return la_product<T, false, false>(a, dtype, ws, ws_bytes, st);
}

struct GradSizes { size_t dz, part, dx, dw, all; };
GradSizes la_grad_sizes(long long M, long long N, long long K, int dtype, int has_slope, int want) {
  GradSizes g{};
  const size_t es = dtype == PN2_DT_F32 ? 4 : 2;
  g.dz = has_slope ? la_align((size_t)M * N * es) : 0;
  g.part = (want & 4) ? la_align((size_t)la_div(M, la_strip(M)) * N * 4) : 0;
  g.dx = (want & 1) ? la_product_bytes(M, K, N, dtype) : 0;
  g.dw = (want & 2) ? la_product_bytes(N, K, M, dtype) : 0;
  g.all = g.dz + g.part + (g.dx > g.dw ? g.dx : g.dw);      // the two products share their partial sums' space, one after the other
  return g;
}

template <class T>
int la_backward(long long M, long long N, long long K, int dtype, const void *dy, long long ldy, const void *slope, const void *x,
                long long ldx, const void *w, long long ldw, void *dx, void *dw, void *db, int db_f32, void *ws, size_t ws_bytes,
                hipStream_t st) {
  const int want = (dx ? 1 : 0) | (dw ? 2 : 0) | (db ? 4 : 0);
  const GradSizes g = la_grad_sizes(M, N, K, dtype, slope != nullptr, want);
  if (ws_bytes < g.all) return PN2_ENOSPC;
  if (g.all && !ws) return PN2_ENULL;
  char *at = (char *)ws;
  void *dz = slope ? at : nullptr;
  float *part = db ? (float *)(at + g.dz) : nullptr;
  char *rest = at + g.dz + g.part;
  const size_t rest_bytes = ws_bytes - g.dz - g.part;
  if (slope || db) {
    const long long strip = la_strip(M), strips = la_div(M, strip);
    la_dz_kernel<T><<<dim3((unsigned)la_div(N, 256), (unsigned)strips), 256, 0, st>>>(M, N, strip, dy, ldy, slope, dz, part);
    if (db) la_db_kernel<T><<<(unsigned)la_div(N, 256), 256, 0, st>>>(N, strips, part, db, db_f32);
    const int rc = pn2_check_launch();
    if (rc != PN2_OK) return rc;
  }
  const void *z = slope ? dz : dy;
  const long long ldz = slope ? N : ldy;
  if (dx) {
    Product a{};
    a.M = M; a.N = K; a.K = N; a.p = z; a.ldp = ldz; a.q = w; a.ldq = ldw; a.e.y = dx;
    const int rc = la_product<T, false, true>(a, dtype, rest, rest_bytes, st);
    if (rc != PN2_OK) return rc;
  }
  if (dw) {
    Product a{};
    a.M = N; a.N = K; a.K = M; a.p = z; a.ldp = ldz; a.q = x; a.ldq = ldx; a.e.y = dw;
    const int rc = la_product<T, true, true>(a, dtype, rest, rest_bytes, st);
    if (rc != PN2_OK) return rc;
  }
  return PN2_OK;
}

}  // namespace

extern "C" size_t pn2_linear_act_workspace_bytes(long long M, int N, int K, int dtype) {
  if (la_bad(M, N, K, dtype) || M == 0) return 0;
  return la_product_bytes(M, N, K, dtype);
}

extern "C" int pn2_linear_act(long long M, int N, int K, int dtype, const void *x, long long ldx, const void *w, long long ldw,
                              const void *bias, int bias_dtype, int act, const void *residual, long long ldr, void *y, void *slope,
                              void *workspace, size_t workspace_bytes, void *stream) {
  if (la_bad(M, N, K, dtype) || act < ACT_NONE || act > ACT_SILU || ldx < 0 || ldw < 0 || ldr < 0 ||
      (bias && bias_dtype != dtype && bias_dtype != PN2_DT_F32))
    return PN2_EINVAL;
  if (M == 0) return PN2_OK;
  if (!x || !w || !y) return PN2_ENULL;
  Product a{};
  a.M = M; a.N = N; a.K = K; a.p = x; a.ldp = ldx; a.q = w; a.ldq = ldw;
  a.e.bias = bias; a.e.bias_f32 = bias_dtype == PN2_DT_F32; a.e.act = act; a.e.res = residual; a.e.ldr = ldr; a.e.y = y;
  a.e.slope = act == ACT_NONE ? nullptr : slope;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == PN2_DT_F32) return la_forward<HdF32>(a, dtype, workspace, workspace_bytes, st);
  if (dtype == PN2_DT_BF16) return la_forward<HdBF16>(a, dtype, workspace, workspace_bytes, st);
  return la_forward<HdF16>(a, dtype, workspace, workspace_bytes, st);
}

extern "C" size_t pn2_linear_act_grad_workspace_bytes(long long M, int N, int K, int dtype, int has_slope, int want) {
  if (la_bad(M, N, K, dtype) || M == 0) return 0;
  return la_grad_sizes(M, N, K, dtype, has_slope, want).all;
}

extern "C" int pn2_linear_act_grad(long long M, int N, int K, int dtype, const void *dy, long long ldy, const void *slope,
                                   const void *x, long long ldx, const void *w, long long ldw, void *dx, void *dw, void *db,
                                   int db_dtype, void *workspace, size_t workspace_bytes, void *stream) {
  if (la_bad(M, N, K, dtype) || M < 1 || ldy < 0 || ldx < 0 || ldw < 0 || (db && db_dtype != dtype && db_dtype != PN2_DT_F32))
    return PN2_EINVAL;
  if (!dy || (dx && !w) || (dw && !x)) return PN2_ENULL;
  hipStream_t st = (hipStream_t)stream;
  const int f32 = db_dtype == PN2_DT_F32;
  if (dtype == PN2_DT_F32) return la_backward<HdF32>(M, N, K, dtype, dy, ldy, slope, x, ldx, w, ldw, dx, dw, db, f32, workspace, workspace_bytes, st);
  if (dtype == PN2_DT_BF16) return la_backward<HdBF16>(M, N, K, dtype, dy, ldy, slope, x, ldx, w, ldw, dx, dw, db, f32, workspace, workspace_bytes, st);
  return la_backward<HdF16>(M, N, K, dtype, dy, ldy, slope, x, ldx, w, ldw, dx, dw, db, f32, workspace, workspace_bytes, st);
}
