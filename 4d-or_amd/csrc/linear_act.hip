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

// act(z) and its slope.  FAST (16-bit results): erf by Abramowitz and Stegun 7.1.26 (|error| <= 1.5e-7, half a step of fp32 where
// it counts), which shares its exponential with the slope; erff costs twice the instructions.
template <int ACT, bool FAST>
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
    const float e = hd_exp2(-0.5f * kHdLog2e * (z * z));
    if constexpr (FAST) {
      // tail = (1 - erf(|z| / sqrt 2)) / 2 = e w:  act = max(z, 0) - |z| tail,  slope = [z > 0] + sign(z) (|z| pdf - tail)
      const float m = fminf(fabsf(z), 1e30f), t = __builtin_amdgcn_rcpf(__fmaf_rn(0.3275911f * 0.7071067811865476f, m, 1.f));
      float w = __fmaf_rn(0.5f * 1.061405429f, t, 0.5f * -1.453152027f);
      w = __fmaf_rn(w, t, 0.5f * 1.421413741f);
      w = __fmaf_rn(w, t, 0.5f * -0.284496736f);
      w = __fmaf_rn(w, t, 0.5f * 0.254829592f);
      w *= t;
      y = __fmaf_rn(-m, e * w, z <= 0.f ? 0.f : z);    // (NaN stays NaN)
      const float h = e * __fmaf_rn(0.3989422804014327f, m, -w);
      d = z > 0.f ? 1.f + h : -h;
    } else {
      const float cdf = __fmaf_rn(0.5f, erff(z * 0.7071067811865476f), 0.5f);
      y = z * cdf;
      d = __fmaf_rn(z * 0.3989422804014327f, e, cdf);
    }
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
  constexpr bool kFast = sizeof(elem) == 2;
  z += la_bias<T>(e, j);
  float y, d;
  switch (e.act) {
    case ACT_RELU: la_act<ACT_RELU, kFast>(z, y, d); break;
    case ACT_GELU: la_act<ACT_GELU, kFast>(z, y, d); break;
    case ACT_GELU_TANH: la_act<ACT_GELU_TANH, kFast>(z, y, d); break;
    case ACT_SILU: la_act<ACT_SILU, kFast>(z, y, d); break;
    default: la_act<ACT_NONE, kFast>(z, y, d);
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
  __device__ __forceinline__ void fetch(const elem *g, long long ld, long long r0, long long R, long long k0, long long k1,
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
    if (n >= VE) {
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
  lp.fetch((const elem *)a.p, a.ldp, i0, a.M, k0, k1, tid);
  lq.fetch((const elem *)a.q, a.ldq, j0, a.N, k0, k1, tid);
  for (long long k = k0; k < k1; k += KB) {
    lp.store(sp, tid);
    lq.store(sq, tid);
    __syncthreads();
    if (k + KB < k1) {
      lp.fetch((const elem *)a.p, a.ldp, i0, a.M, k + KB, k1, tid);
      lq.fetch((const elem *)a.q, a.ldq, j0, a.N, k + KB, k1, tid);
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

// ------------------------------------------------------------------------------------------------------ the tile kernel
// A workgroup of WI x WJ waves owns a tile of (WI TI 16) x (WJ TJ 16) results; a wave holds TI x TJ accumulators.  Operand tiles of
// 128 bytes of contraction (64 16-bit or 32 fp32 indices: whole cache lines of a K operand, whose 64-byte halves cost the L1 twice
// the requests) travel global -> LDS directly (global_load_lds, 16 bytes per lane) into one of two slots, a tile ahead.  A tile is
// two steps; the fragments of a step are read from LDS while the matrix instructions of the step before run, so a wave never waits
// for LDS, and there is one barrier per tile.
//
// LDS layout (16-byte pieces; XOR swizzles, applied to the GLOBAL address of a lane because the direct load writes lane-linear):
//   K operand: rows of 128 bytes, piece c of row r at c ^ f(r), f counting the fragment's row pairs: a ds_read_b128 takes 16 lanes
//     per cycle, {0-3, 12-15, 20-23, 24-27} and so on, and those hit the 16 pieces of 256 bytes;
//   R operand: contraction rows of the tile's columns, piece c of row k at c ^ f(k); 16-bit fragments are read with the
//     transposing ds_read_b64_tr_b16 (lane 4 b + a of 16 gives row b, columns 4 a .. 4 a + 3 and receives column lane, rows 0 .. 3),
//     fp32 ones element by element.
// Q's fragments are a permutation of its rows: fragment u, row r is j = (u >> 1) 32 + (r >> 2) 8 + (u & 1) 4 + (r & 3) of a group of
// 64, so that two fragments give a lane 8 consecutive columns, and the four lanes of a row 32: 64 whole bytes per row and store.
template <int V> struct LaInt { static constexpr int value = V; };
template <int N, int I = 0, class F>
__device__ __forceinline__ void la_each(F f) {
  if constexpr (I < N) {
    f(LaInt<I>{});
    la_each<N, I + 1>(f);
  }
}

__device__ __forceinline__ unsigned la_lds(const void *p) {
  return (unsigned)(size_t)(__attribute__((address_space(3))) const char *)p;
}
// 64 lanes x 16 bytes, global (uniform base + lane offset) -> LDS (uniform base + 16 lane)
__device__ __forceinline__ void la_dma(unsigned lds, unsigned long long base, unsigned off) {
  // (inline asm: the builtin is counted into lgkmcnt too, and every ds_read would wait for it; awaited by la_wait)
  unsigned keep;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %3\n\ts_mov_b32 m0, %0"
               : "=&s"(keep) : "s"(lds), "v"(off), "s"(base) : "memory");
}
// all but the last N direct loads of this wave have landed, its LDS reads are done
template <int N>
__device__ __forceinline__ void la_wait() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}

template <bool PERM>
__device__ __forceinline__ int la_swz_k(int r) {
  return PERM ? ((r >> 1) & 1) | ((r >> 2) & 6) : (r >> 1) & 7;
}
template <bool PERM>
__device__ __forceinline__ int la_swz_r(int k) {
  return PERM ? (k & 3) << 2 : ((k & 3) << 1) | (k & 8);
}

template <class T, bool ROWS, bool PERM, int B, int NT>
struct Operand {
  typedef typename T::elem elem;
  static constexpr int VE = T::kPerVec, KB = 8 * VE, ES = (int)sizeof(elem), PER = B * 8 / NT;   // pieces per thread and tile
  static constexpr int PW = B / VE;                                                              // R operand: pieces per row
  unsigned off[PER];               // lane offsets of the direct loads
  unsigned long long base;         // advances by a tile
  unsigned step;
  __device__ __forceinline__ void init(const void *g, long long ld, long long r0, long long R, long long k0, int tid) {
    const elem *p = (const elem *)g;
    base = (unsigned long long)(ROWS ? p + k0 * ld + r0 : p + r0 * ld + k0);
    step = ROWS ? (unsigned)(KB * ld * ES) : 128u;
#pragma unroll
    for (int n = 0; n < PER; ++n) {
      const int at = n * NT + tid;
      if constexpr (!ROWS) {
        const int r = at >> 3, c = (at & 7) ^ la_swz_k<PERM>(r);
        const long long rr = r0 + r < R ? r : R - 1 - r0;          // rows out of range repeat the last one: never stored
        off[n] = (unsigned)(rr * ld * ES + c * 16);
      } else {
        const int k = at / PW, c = (at % PW) ^ la_swz_r<PERM>(k);
        const long long cc = r0 + (long long)(c + 1) * VE <= R ? c * VE : R - VE - r0;
        off[n] = (unsigned)(k * ld * ES + cc * ES);
      }
    }
  }
  __device__ __forceinline__ void issue(int n, unsigned lds, int wave) { la_dma(lds + (n * NT + wave * 64) * 16, base, off[n]); }
  // the last, partial tile: pieces through registers, out of range = 0
  __device__ __forceinline__ void tail(char *lds, const void *g, long long ld, long long r0, long long R, long long k0, long long k1,
                                       int tid) {
#pragma unroll
    for (int n = 0; n < PER; ++n) {
      const int at = n * NT + tid;
      long long r, k, left;
      if constexpr (!ROWS) {
        r = r0 + (at >> 3);
        k = k0 + ((at & 7) ^ la_swz_k<PERM>(at >> 3)) * VE;
        left = r < R ? k1 - k : 0;
      } else {
        k = k0 + at / PW;
        r = r0 + ((at % PW) ^ la_swz_r<PERM>(at / PW)) * VE;
        left = k < k1 ? R - r : 0;
      }
      const elem *src = (const elem *)g + (ROWS ? k * ld + r : r * ld + k);
      hd_u32x4 w = {0, 0, 0, 0};
      if (left >= VE) {
        w = hd_load16<T>(src);
      } else {
        elem v[VE];
#pragma unroll
        for (int i = 0; i < VE; ++i) v[i] = i < left ? src[i] : T::round(0.f);
        __builtin_memcpy(&w, v, 16);
      }
      *reinterpret_cast<hd_u32x4 *>(lds + at * 16) = w;
    }
  }
  // Fragment t, step `half` of the tile, of the wave whose rows start at w0 (a multiple of 64) = frag(slot + lane_base(w0), t, half):
  // a lane's offsets differ between fragments by a constant, or by a constant exclusive-or.
  __device__ __forceinline__ static unsigned lane_base(int w0, int lane) {
    const int r = lane & 15, g = lane >> 4;
    if constexpr (!ROWS) {
      const int row = w0 + (PERM ? (r >> 2) * 8 + (r & 3) : r);            // (its swizzle does not depend on t)
      return row * 128 + ((g ^ la_swz_k<PERM>(row)) << 4);
    } else if constexpr (ES == 2) {
      const int a = r & 3, k = g * 8 + (r >> 2), col = w0 + a * (PERM ? 8 : 4);
      return k * (B * 2) + (((col >> 3) ^ la_swz_r<PERM>(k)) << 4) + ((col >> 2) & 1) * 8;
    } else {
      return w0 + (PERM ? (r >> 2) * 8 + (r & 3) : r);                     // (the column; fp32 pays the address of every element)
    }
  }
  template <int HALF>
  __device__ __forceinline__ static hd_u32x4 frag(unsigned slot, unsigned base, int t, int lane) {
    typedef __attribute__((address_space(3))) const hd_u32x4 *lds16;
    if constexpr (!ROWS) {
      return *(lds16)(size_t)(((slot + base) ^ (HALF << 6)) + (PERM ? (t >> 1) * 4096 + (t & 1) * 512 : t * 2048));
    } else if constexpr (ES == 2) {
      typedef short s4 __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) s4 *lds8;
      // natural: 16 columns are 2 pieces;  permuted: 32 columns are 4 pieces, 4 columns half a piece
      const unsigned at = ((slot + base) ^ (PERM ? (t >> 1) << 6 : t << 5)) + HALF * 32 * B * 2 + (PERM ? (t & 1) * 8 : 0);
      const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds8)(size_t)at);
      const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds8)(size_t)(at + 4 * B * 2));      // four rows on: the same swizzle
      return __builtin_bit_cast(hd_u32x4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      const int col = (int)base + (PERM ? (t >> 1) * 32 + (t & 1) * 4 : t * 16);
      hd_u32x4 w;
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const int k = HALF * 16 + (lane >> 4) * 4 + n;
        w[n] = *(__attribute__((address_space(3))) const unsigned *)(size_t)(slot + k * (B * 4) + (((col >> 2) ^ la_swz_r<PERM>(k)) << 4) + (col & 3) * 4);
      }
      return w;
    }
  }
};

// 8 consecutive elements; FULL: all of them in range, otherwise the first `left` (the others 0)
template <class T, bool FULL>
__device__ __forceinline__ void la_load8(const typename T::elem *p, long long left, float (&f)[8]) {
  if (FULL || left >= 8) {
    if constexpr (T::kPerVec == 8) {
      T::unpack(hd_load16<T>(p), f);
    } else {
      float lo[4], hi[4];
      T::unpack(hd_load16<T>(p), lo);
      T::unpack(hd_load16<T>(p + 4), hi);
#pragma unroll
      for (int n = 0; n < 4; ++n) { f[n] = lo[n]; f[4 + n] = hi[n]; }
    }
  } else {
#pragma unroll
    for (int n = 0; n < 8; ++n) f[n] = n < left ? T::load(p + n) : 0.f;
  }
}
template <class T, bool FULL>
__device__ __forceinline__ void la_store8(typename T::elem *p, long long left, const float (&f)[8]) {
  if (FULL || left >= 8) {
    if constexpr (T::kPerVec == 8) {
      hd_store16<T>(p, T::pack(f));
    } else {
      float lo[4] = {f[0], f[1], f[2], f[3]}, hi[4] = {f[4], f[5], f[6], f[7]};
      hd_store16<T>(p, T::pack(lo));
      hd_store16<T>(p + 4, T::pack(hi));
    }
  } else {
#pragma unroll
    for (int n = 0; n < 8; ++n)
      if (n < left) p[n] = T::round(f[n]);
  }
}

// The accumulators of a wave (its first row i, its lane's first column j) -> results.  A lane's columns are runs of 8 at
// j + 16 u, u even.  FULL: the tile lies inside the matrix (no guards).  The bias of all columns and the residual
// of two rows at a time are read before the stores (loads between stores would wait for each other).
template <class T, int ACT, bool FULL, bool RES, int TI, int TJ>
__device__ __forceinline__ void la_epilogue(const Product &a, const la_f32x4 (&acc)[TI][TJ], long long i, long long j) {
  typedef typename T::elem elem;
  typedef typename SlopeOf<T>::type S;
  const Epilogue &e = a.e;
  auto col = [&](int u) { return j + u * 16; };
  float b[TJ / 2][8];
#pragma unroll
  for (int u = 0; u < TJ; u += 2) {
#pragma unroll
    for (int n = 0; n < 8; ++n) b[u / 2][n] = 0.f;
    if (e.bias) {
      if (e.bias_f32) la_load8<HdF32, FULL>((const float *)e.bias + col(u), a.N - col(u), b[u / 2]);
      else la_load8<T, FULL>((const elem *)e.bias + col(u), a.N - col(u), b[u / 2]);
    }
  }
  // (static indices by construction: as a loop, the long body is unrolled too late for the accumulators to stay in registers)
  la_each<TI / 2>([&](auto g_) __attribute__((always_inline)) {
    constexpr int t0 = decltype(g_)::value * 2;
    float r[2][TJ / 2][8];
    if constexpr (RES) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int u = 0; u < TJ; u += 2) {
          const long long row = i + (t0 + t) * 16;
          la_load8<T, FULL>((const elem *)e.res + row * e.ldr + col(u), FULL || row < a.M ? a.N - col(u) : 0, r[t][u / 2]);
        }
    }
    la_each<TJ>([&](auto n_) __attribute__((always_inline)) {
      constexpr int t = decltype(n_)::value / (TJ / 2), u = decltype(n_)::value % (TJ / 2) * 2;
      const long long row = i + (t0 + t) * 16, left = FULL || row < a.M ? a.N - col(u) : 0;
      if (!FULL && left <= 0) return;
      float y[8], d[8];
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        la_act<ACT, sizeof(elem) == 2>(acc[t0 + t][u + n / 4][n % 4] + b[u / 2][n], y[n], d[n]);
        if constexpr (RES) y[n] += r[t][u / 2][n];
      }
      la_store8<T, FULL>((elem *)e.y + row * a.N + col(u), left, y);
      if constexpr (ACT != ACT_NONE) {
        if (e.slope) la_store8<S, FULL>((typename S::elem *)e.slope + row * a.N + col(u), left, d);
      }
    });
  });
}

// ... -> the partial sums of a split contraction
template <int TI, int TJ>
__device__ __forceinline__ void la_partial(const Product &a, const la_f32x4 (&acc)[TI][TJ], long long i, long long j) {
  la_each<TI * TJ / 2>([&](auto n_) __attribute__((always_inline)) {
    constexpr int t = decltype(n_)::value / (TJ / 2), u = decltype(n_)::value % (TJ / 2) * 2;
    const long long row = i + t * 16, c = j + u * 16, left = row < a.M ? a.N - c : 0;
    if (left <= 0) return;
    float y[8];
#pragma unroll
    for (int n = 0; n < 8; ++n) y[n] = acc[t][u + n / 4][n % 4];
    la_store8<HdF32, false>(a.partial + ((long long)blockIdx.z * a.M + row) * a.N + c, left, y);
  });
}

template <class T, bool PROWS, bool QROWS, int WI, int WJ, int TI, int TJ, int ACT>
__global__ __launch_bounds__(64 * WI * WJ, 2) void la_tile_kernel(Product a, int gi, int gj) {
  constexpr int NT = 64 * WI * WJ, BI = WI * TI * 16, BJ = WJ * TJ * 16, KB = 8 * T::kPerVec, SLOT = (BI + BJ) * 128;
  typedef Operand<T, PROWS, false, BI, NT> OP;
  typedef Operand<T, QROWS, true, BJ, NT> OQ;
  __shared__ __align__(1024) char ring[2 * SLOT];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // workgroups go round robin over the 8 XCDs: give each XCD a contiguous run of tiles, walked in bands of 8 tile rows, so that the
  // operand panels of a band are shared in its L2
  int ti, tj;
  {
    const int n = gi * gj, id = blockIdx.x, per = n / 8, rem = n % 8, x = id % 8, q = id / 8;
    const int at = x * per + (x < rem ? x : rem) + q;
    const int band = at / (8 * gj), rows = gi - band * 8 < 8 ? gi - band * 8 : 8, in = at - band * 8 * gj;
    ti = band * 8 + in % rows;
    tj = in / rows;
  }
  const long long i0 = (long long)ti * BI, j0 = (long long)tj * BJ;
  const long long k0 = (long long)blockIdx.z * a.kchunk, k1 = k0 + a.kchunk < a.K ? k0 + a.kchunk : a.K;
  const int tiles = (int)((k1 - k0) / KB), rest = (int)((k1 - k0) % KB);
  const int wi = (wave % WI) * TI * 16, wj = (wave / WI) * TJ * 16;
  constexpr int L = OP::PER + OQ::PER;                 // direct loads per wave and tile
  OP op;
  OQ oq;
  op.init(a.p, a.ldp, i0, a.M, k0, tid);
  oq.init(a.q, a.ldq, j0, a.N, k0, tid);
  const unsigned lds0 = la_lds(ring);
  // direct load n of the next tile; beyond the last tile it repeats that one (in bounds, into a slot nobody reads any more), so that
  // the loop has no branches and its waits are constants
  int issued = 0;
  auto issue = [&](int n) __attribute__((always_inline)) {
    const unsigned at = __builtin_amdgcn_readfirstlane(lds0 + (issued & 1) * SLOT);
    if (n < OP::PER) op.issue(n, at, wave);
    else oq.issue(n - OP::PER, at + BI * 128, wave);
    if (n == L - 1) {
      ++issued;
      op.base += issued < tiles ? op.step : 0;
      oq.base += issued < tiles ? oq.step : 0;
    }
  };
  la_f32x4 acc[TI][TJ] = {};
  hd_u32x4 p[2][TI], q[2][TJ];
  const unsigned pb = OP::lane_base(wi, lane), qb = OQ::lane_base(wj, lane);
  // fragment n of step HALF of the tile in `slot`, Q's first -> register set HALF
  auto read = [&](unsigned slot, int n, auto half_) __attribute__((always_inline)) {
    constexpr int half = decltype(half_)::value;
    if (n < TJ) q[half][n] = OQ::template frag<half>(slot + BI * 128, qb, n, lane);
    else p[half][n - TJ] = OP::template frag<half>(slot, pb, n - TJ, lane);
  };
  // A step: the products of register set HALF, one read of the other set's fragments after every GAP of the first ones, LOAD: the
  // direct loads in between, in its first half (they have little more than a step to land).  The order is pinned: left to itself the compiler sinks the reads, and the next step waits for them;
  // loads before the products leave the matrix cores idle behind the barrier.
  constexpr int GAP = TI * TJ * 3 / 4 / (TI + TJ), LGAP = TI * TJ / L / 2 > 0 ? TI * TJ / L / 2 : 1;
  static_assert(GAP > 0 && LGAP > 0, "room for the reads and the loads between the products");
  auto step = [&](unsigned slot, auto half_, auto load_) __attribute__((always_inline)) {
    constexpr int half = decltype(half_)::value;
    la_each<TI * TJ>([&](auto n_) __attribute__((always_inline)) {
      constexpr int n = decltype(n_)::value, t = n / TJ, u = n % TJ;
      acc[t][u] = la_mma(T{}, q[half][u], p[half][t], acc[t][u]);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (n % GAP == 0 && n / GAP < TI + TJ) read(slot, n / GAP, LaInt<half ^ 1>{});
      if constexpr (decltype(load_)::value && n % LGAP == LGAP / 2 && n / LGAP < L) issue(n / LGAP);
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  // every wave's direct loads have landed (all but the last N of each) and its LDS reads are done
  auto meet = [&](auto n_) __attribute__((always_inline)) {
    la_wait<decltype(n_)::value>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  if (tiles > 0) {
#pragma unroll
    for (int n = 0; n < 2 * L; ++n) issue(n % L);
    meet(LaInt<L>{});
#pragma unroll
    for (int n = 0; n < TI + TJ; ++n) read(lds0, n, LaInt<0>{});
    for (int d = 0; d < tiles; ++d) {
      step(lds0 + (d & 1) * SLOT, LaInt<0>{}, LaInt<0>{});
      // the next tile has landed; this one's slot, whose last fragments were read in the step above, is refilled
      meet(LaInt<0>{});
      // (the last tile reads on in a slot of older data: in bounds, never used)
      step(lds0 + ((d + 1) & 1) * SLOT, LaInt<1>{}, LaInt<1>{});
    }
    la_wait<0>();                                      // no direct load is left when the workgroup gives its LDS back
  }
  if (rest) {
    __syncthreads();
    op.tail(ring, a.p, a.ldp, i0, a.M, k0 + (long long)tiles * KB, k1, tid);
    oq.tail(ring + BI * 128, a.q, a.ldq, j0, a.N, k0 + (long long)tiles * KB, k1, tid);
    __syncthreads();
    auto half = [&](auto half_) __attribute__((always_inline)) {
      constexpr int h = decltype(half_)::value;
#pragma unroll
      for (int n = 0; n < TI + TJ; ++n) read(lds0, n, LaInt<h>{});
#pragma unroll
      for (int t = 0; t < TI; ++t)
#pragma unroll
        for (int u = 0; u < TJ; ++u) acc[t][u] = la_mma(T{}, q[h][u], p[h][t], acc[t][u]);
    };
    half(LaInt<0>{});
    if (rest > KB / 2) half(LaInt<1>{});
  }
  const long long i = i0 + wi + (lane & 15), j = j0 + wj + (lane >> 4) * 8;
  if (a.splits > 1) la_partial(a, acc, i, j);
  else if (i0 + BI > a.M || j0 + BJ > a.N) {
    if (a.e.res) la_epilogue<T, ACT, false, true>(a, acc, i, j);
    else la_epilogue<T, ACT, false, false>(a, acc, i, j);
  } else {
    if (a.e.res) la_epilogue<T, ACT, true, true>(a, acc, i, j);
    else la_epilogue<T, ACT, true, false>(a, acc, i, j);
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

// dz = dy slope (SLOPE; otherwise dz is dy itself) and column sums: a workgroup takes 64 x VE columns and a strip of rows, its four
// waves every fourth row; part (strips, N) fp32, or NULL.  Bound by its bytes (read dy and slope, write dz).
template <class T, bool SLOPE>
__global__ __launch_bounds__(256) void la_dz_kernel(long long M, long long N, int strip, const void *dy_, long long ldy,
                                                    const void *slope_, void *dz_, float *part) {
  typedef typename T::elem elem;
  typedef typename SlopeOf<T>::type S;
  constexpr int VE = T::kPerVec, U = 4;
  __shared__ float sum[3][64][VE];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long long j = ((long long)blockIdx.x * 64 + lane) * VE, left = N - j;
  const long long i0 = (long long)blockIdx.y * strip, i1 = i0 + strip < M ? i0 + strip : M;
  float s[VE];
#pragma unroll
  for (int n = 0; n < VE; ++n) s[n] = 0.f;
  if (left >= VE) {
    const elem *dy = (const elem *)dy_ + j;
    const typename S::elem *slope = (const typename S::elem *)slope_ + j;
    elem *dz = (elem *)dz_ + j;
    for (long long i = i0 + wave; i < i1; i += 4 * U) {
      hd_u32x4 wy[U], ws[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const long long row = i + 4 * u < i1 ? i + 4 * u : i;              // (a row past the strip repeats the first)
        wy[u] = hd_load16<T>(dy + row * ldy);
        if constexpr (SLOPE) ws[u] = hd_load16<S>(slope + row * N);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (i + 4 * u >= i1) break;
        float f[VE];
        T::unpack(wy[u], f);
        if constexpr (SLOPE) {
          float d[VE];
          S::unpack(ws[u], d);
#pragma unroll
          for (int n = 0; n < VE; ++n) f[n] *= d[n];
          hd_store16<T>(dz + (i + 4 * u) * N, T::pack(f));
        }
#pragma unroll
        for (int n = 0; n < VE; ++n) s[n] += f[n];
      }
    }
  } else if (left > 0) {
    for (long long i = i0 + wave; i < i1; i += 4)
#pragma unroll
      for (int n = 0; n < VE; ++n) {
        if (n >= left) continue;
        float f = T::load((const elem *)dy_ + i * ldy + j + n);
        if constexpr (SLOPE) {
          f *= S::load((const typename S::elem *)slope_ + i * N + j + n);
          ((elem *)dz_)[i * N + j + n] = T::round(f);
        }
        s[n] += f;
      }
  }
  if (!part) return;                                   // uniform
  if (wave) {
#pragma unroll
    for (int n = 0; n < VE; ++n) sum[wave - 1][lane][n] = s[n];
  }
  __syncthreads();
  if (wave == 0) {
#pragma unroll
    for (int n = 0; n < VE; ++n)
      if (n < left) part[(long long)blockIdx.y * N + j + n] = (s[n] + sum[0][lane][n]) + (sum[1][lane][n] + sum[2][lane][n]);
  }
}

// the strips' sums joined: 64 columns per workgroup, its four waves every fourth strip
template <class T>
__global__ __launch_bounds__(256) void la_db_kernel(long long N, int strips, const float *part, void *db, int db_f32) {
  __shared__ float sum[3][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long long j = (long long)blockIdx.x * 64 + lane;
  float s = 0.f;
  if (j < N)
    for (int i = wave; i < strips; i += 4) s += part[(long long)i * N + j];
  if (wave) sum[wave - 1][lane] = s;
  __syncthreads();
  if (wave || j >= N) return;
  s = (s + sum[0][lane]) + (sum[1][lane] + sum[2][lane]);
  if (db_f32) ((float *)db)[j] = s;
  else ((typename T::elem *)db)[j] = T::round(s);
}

constexpr long long kMaxDim = 1LL << 31;

inline long long la_div(long long a, long long b) { return (a + b - 1) / b; }
inline size_t la_align(size_t n) { return (n + 255) & ~(size_t)255; }

// Which kernel a product takes, by size, type and alignment, and how often its contraction is split.
//   big   (256 x 256, 16-bit only): tiles for at least three quarters of the CUs.  8192^3: 1.35-1.46 PFLOP/s against 0.88 for mid
//   mid   (128 x 128, two workgroups per CU)
//   any   (64 x 64): one side below 96, or operands whose rows are no 16-byte pieces
// A contraction is split until two workgroups per CU run, each at least four steps long.
enum { KERNEL_ANY, KERNEL_MID, KERNEL_BIG };

bool la_vec(const void *p, long long ld, int dtype) {
  const long long es = dtype == PN2_DT_F32 ? 4 : 2;
  return ((uintptr_t)p & 15) == 0 && (ld * es) % 16 == 0 && ld <= (1 << 22);
}

int la_kernel_for(long long M, long long N, long long K, int dtype) {           // by size alone
  if (M < 96 || N < 96 || K < (dtype == PN2_DT_F32 ? 16 : 32)) return KERNEL_ANY;
  return dtype != PN2_DT_F32 && la_div(M, 256) * la_div(N, 256) >= 192 ? KERNEL_BIG : KERNEL_MID;
}

// the tile kernels' direct loads need 16-byte pieces: aligned bases and strides, and axes that are whole pieces
bool la_pieces(const Product &a, int dtype, bool prows, bool qrows) {
  const long long ve = dtype == PN2_DT_F32 ? 4 : 8;
  return la_vec(a.p, a.ldp, dtype) && la_vec(a.q, a.ldq, dtype) && (prows ? a.M : a.K) % ve == 0 && (qrows ? a.N : a.K) % ve == 0;
}

// -> contraction indices per split
long long la_chunk(long long M, long long N, long long K, int dtype, int kernel) {
  const long long kb = dtype == PN2_DT_F32 ? 32 : 64, steps = la_div(K, kb);
  const long long edge = kernel == KERNEL_BIG ? 256 : kernel == KERNEL_MID ? 128 : 64;
  long long s = (kernel == KERNEL_BIG ? 256 : 512) / (la_div(M, edge) * la_div(N, edge));
  if (s > steps / 2) s = steps / 2;
  if (s < 1) s = 1;
  if (s > 64) s = 64;
  return la_div(steps, s) * kb;
}

size_t la_partial_bytes(long long M, long long N, long long K, int dtype, int kernel) {
  const long long splits = la_div(K, la_chunk(M, N, K, dtype, kernel));
  return splits > 1 ? la_align((size_t)splits * M * N * 4) : 0;
}

// the most a product of this size can need, whatever its operands' alignment
size_t la_product_bytes(long long M, long long N, long long K, int dtype) {
  const size_t any = la_partial_bytes(M, N, K, dtype, KERNEL_ANY), tile = la_partial_bytes(M, N, K, dtype, la_kernel_for(M, N, K, dtype));
  return any > tile ? any : tile;
}

template <class T, bool PROWS, bool QROWS, int WI, int WJ, int TI, int TJ>
int la_tile_as(const Product &a, hipStream_t st) {
  const int gi = (int)la_div(a.M, WI * TI * 16), gj = (int)la_div(a.N, WJ * TJ * 16);
  const dim3 grid((unsigned)(gi * gj), 1, (unsigned)a.splits);
  constexpr int NT = 64 * WI * WJ;
  if constexpr (PROWS || QROWS) {
    la_tile_kernel<T, PROWS, QROWS, WI, WJ, TI, TJ, ACT_NONE><<<grid, NT, 0, st>>>(a, gi, gj);
  } else {
    switch (a.splits > 1 ? ACT_NONE : a.e.act) {       // (a split contraction's epilogue is the join kernel's)
      case ACT_RELU: la_tile_kernel<T, false, false, WI, WJ, TI, TJ, ACT_RELU><<<grid, NT, 0, st>>>(a, gi, gj); break;
      case ACT_GELU: la_tile_kernel<T, false, false, WI, WJ, TI, TJ, ACT_GELU><<<grid, NT, 0, st>>>(a, gi, gj); break;
      case ACT_GELU_TANH: la_tile_kernel<T, false, false, WI, WJ, TI, TJ, ACT_GELU_TANH><<<grid, NT, 0, st>>>(a, gi, gj); break;
      case ACT_SILU: la_tile_kernel<T, false, false, WI, WJ, TI, TJ, ACT_SILU><<<grid, NT, 0, st>>>(a, gi, gj); break;
      default: la_tile_kernel<T, false, false, WI, WJ, TI, TJ, ACT_NONE><<<grid, NT, 0, st>>>(a, gi, gj);
    }
  }
  if (a.splits > 1) la_join_kernel<T><<<(unsigned)la_div(a.M * a.N, 256), 256, 0, st>>>(a);
  return pn2_check_launch();
}

template <class T, bool PROWS, bool QROWS>
int la_product(Product a, int dtype, void *ws, size_t ws_bytes, hipStream_t st) {
  const int kernel = la_pieces(a, dtype, PROWS, QROWS) ? la_kernel_for(a.M, a.N, a.K, dtype) : KERNEL_ANY;
  a.kchunk = la_chunk(a.M, a.N, a.K, dtype, kernel);
  a.splits = (int)la_div(a.K, a.kchunk);
  const size_t need = la_partial_bytes(a.M, a.N, a.K, dtype, kernel);
  if (ws_bytes < need) return PN2_ENOSPC;
  if (need && !ws) return PN2_ENULL;
  a.partial = (float *)ws;
  if constexpr (sizeof(typename T::elem) == 2) {
    if (kernel == KERNEL_BIG) return la_tile_as<T, PROWS, QROWS, 2, 4, 8, 4>(a, st);
  }
  if (kernel != KERNEL_ANY) return la_tile_as<T, PROWS, QROWS, 2, 2, 4, 4>(a, st);
  const long long gx = la_div(a.M, 64), gy = la_div(a.N, 64);
  if (gy > 65535) return PN2_EINVAL;
  la_any_kernel<T, PROWS, QROWS><<<dim3((unsigned)gx, (unsigned)gy, (unsigned)a.splits), 256, 0, st>>>(a);
  if (a.splits > 1) la_join_kernel<T><<<(unsigned)la_div(a.M * a.N, 256), 256, 0, st>>>(a);
  return pn2_check_launch();
}

inline bool la_bad(long long M, long long N, long long K, int dtype) {
  return M < 0 || N < 1 || K < 1 || M >= kMaxDim || N > 65535LL * 64 || K > 65535LL * 64 || dtype < PN2_DT_F32 || dtype > PN2_DT_F16;
}

// rows per partial column sum: enough workgroups for the chip, at least 16 rows each, at most 512 strips
inline int la_strip(long long M, long long N, int dtype) {
  const long long cols = la_div(N, dtype == PN2_DT_F32 ? 256 : 512);
  long long strips = la_div(2048, cols);
  if (strips > 512) strips = 512;
  long long s = la_div(M, strips);
  return (int)(s < 16 ? 16 : s);
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
  g.part = (want & 4) ? la_align((size_t)la_div(M, la_strip(M, N, dtype)) * N * 4) : 0;
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
    const int strip = la_strip(M, N, dtype), strips = (int)la_div(M, strip);
    const dim3 grid((unsigned)la_div(N, 64 * T::kPerVec), (unsigned)strips);
    if (slope) la_dz_kernel<T, true><<<grid, 256, 0, st>>>(M, N, strip, dy, ldy, slope, dz, part);
    else la_dz_kernel<T, false><<<grid, 256, 0, st>>>(M, N, strip, dy, ldy, nullptr, nullptr, part);
    if (db) la_db_kernel<T><<<(unsigned)la_div(N, 64), 256, 0, st>>>(N, strips, part, db, db_f32);
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
