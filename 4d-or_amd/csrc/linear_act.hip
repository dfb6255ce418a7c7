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
// in 16-bit fixed point, steps of 2^-14: off by at most 2^-15 (fp16 would be off by up to 2^-11 near 1, bf16 by 2^-8), 0 and 1
// exact, NaN as -2.  dz is rounded to the operands' type for the matrix cores.
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

// act(z) and its slope.  FAST (16-bit results): erf by Abramowitz and Stegun 7.1.26, which shares its exponential with the slope; erff
// costs twice the instructions.  Off by 1.5e-7 (2.5 u, u = 2^-24) in erf and 2.1e-7 in act(z), absolutely.  Relative to a result that
// goes to zero, far below it: 5e-4 at z = -4 (fp16's half step there is 2.4e-4 to 4.9e-4), 1.6e-3 at -5, 3.6e-3 at -6 (bf16's half
// step: 2e-3 to 3.9e-3), 1 % at -8, where act is 5e-15.  The fp32 form is erff's, whose 1 + erf cancels there: half a step of 1/2 is
// 9e-4 of it at -4 and 10 % at -5.
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
    // (1 + tanh u) / 2 = 1 / (1 + e^(-2u)), u = sqrt(2/pi) (z + 0.044715 z^3); beyond |z| = 30 the gate is 0 or 1 (fminf and fmaxf
    // would turn a NaN into -30, and its slope into 0)
    const float w = z != z ? z : fminf(fmaxf(z, -30.f), 30.f), w2 = w * w;
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
  void *slope;              // (M, N) dense, fp32 for fp32 and fixed point for 16-bit types, or NULL
};

struct Fixed {              // 16-bit fixed point, see above
  typedef short elem;
  static constexpr int kPerVec = 8;
  static __device__ __forceinline__ float value(int i) { return i == -32768 ? __builtin_nanf("") : (float)i * 0x1p-14f; }
  static __device__ __forceinline__ float load(const elem *p) { return value(*p); }
  static __device__ __forceinline__ elem round(float v) { return v == v ? (elem)rintf(v * 0x1p14f) : (elem)-32768; }
  static __device__ __forceinline__ void unpack(hd_u32x4 w, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int u = (int)w[i];
      f[2 * i] = value((short)u);
      f[2 * i + 1] = value(u >> 16);
    }
  }
  static __device__ __forceinline__ hd_u32x4 pack(const float (&f)[8]) {
    hd_u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // two of them in one instruction: round(32767 v)
      typedef short s2 __attribute__((ext_vector_type(2)));
      const s2 h = __builtin_bit_cast(s2, __builtin_amdgcn_cvt_pknorm_i16(f[2 * i] * (16384.f / 32767.f), f[2 * i + 1] * (16384.f / 32767.f)));
      w[i] = __builtin_bit_cast(unsigned, h);
    }
    const float any = ((f[0] + f[1]) + (f[2] + f[3])) + ((f[4] + f[5]) + (f[6] + f[7]));
    if (!(any == any)) {                               // rare
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = (unsigned short)round(f[2 * i]) | (unsigned)(unsigned short)round(f[2 * i + 1]) << 16;
    }
    return w;
  }
};

template <class T> struct SlopeOf { typedef Fixed type; };
template <> struct SlopeOf<HdF32> { typedef HdF32 type; };

struct Product {
  long long M, N, K;
  const void *p, *q;
  long long ldp, ldq;
  long long rp, rq;         // rows of P and Q that may be read (an R operand's padded to whole 16-byte pieces)
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
// PW pieces per row.  A transposing read takes rows k & 3 at once; rows of 8 pieces (128 bytes) alternate between the halves of 256
// bytes by themselves.
template <bool PERM, int PW>
__device__ __forceinline__ int la_swz_r(int k) {
  if constexpr (PW == 8) return PERM ? (k & 2) << 1 : (k & 2) | ((k & 8) >> 1);
  else return PERM ? (k & 3) << 2 : ((k & 3) << 1) | (k & 8);
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
        const int k = at / PW, c = (at % PW) ^ la_swz_r<PERM, PW>(k);
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
        r = r0 + ((at % PW) ^ la_swz_r<PERM, PW>(at / PW)) * VE;
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
  // Fragment t, step `half` of the tile, of the wave whose rows start at w0 (a multiple of 32) = frag(slot + lane_base(w0), t, half):
  // a lane's offsets differ between fragments by a constant, or by a constant exclusive-or.
  __device__ __forceinline__ static unsigned lane_base(int w0, int lane) {
    const int r = lane & 15, g = lane >> 4;
    if constexpr (!ROWS) {
      const int row = w0 + (PERM ? (r >> 2) * 8 + (r & 3) : r);            // (its swizzle does not depend on t)
      return row * 128 + ((g ^ la_swz_k<PERM>(row)) << 4);
    } else if constexpr (ES == 2) {
      const int a = r & 3, k = g * 8 + (r >> 2), col = w0 + a * (PERM ? 8 : 4);
      return k * (B * 2) + (((col >> 3) ^ la_swz_r<PERM, PW>(k)) << 4) + ((col >> 2) & 1) * 8;
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
        w[n] = *(__attribute__((address_space(3))) const unsigned *)(size_t)(slot + k * (B * 4) + (((col >> 2) ^ la_swz_r<PERM, PW>(k)) << 4) + (col & 3) * 4);
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
    la_each<2>([&](auto t_) __attribute__((always_inline)) {
      constexpr int t = decltype(t_)::value;
      const long long row = i + (t0 + t) * 16;
      if (!FULL && row >= a.M) return;
      float y[TJ / 2][8], d[TJ / 2][8];
#pragma unroll
      for (int u = 0; u < TJ; u += 2)
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          la_act<ACT, sizeof(elem) == 2>(acc[t0 + t][u + n / 4][n % 4] + b[u / 2][n], y[u / 2][n], d[u / 2][n]);
          if constexpr (RES) y[u / 2][n] += r[t][u / 2][n];
        }
      // (the halves of a cache line of y one right after the other, then the slope's: between them a line can leave the cache half
      // written, and the tile's results are more than the cache)
#pragma unroll
      for (int u = 0; u < TJ; u += 2)
        if (FULL || a.N > col(u)) la_store8<T, FULL>((elem *)e.y + row * a.N + col(u), a.N - col(u), y[u / 2]);
      if constexpr (ACT != ACT_NONE) {
        if (e.slope) {
#pragma unroll
          for (int u = 0; u < TJ; u += 2)
            if (FULL || a.N > col(u)) la_store8<S, FULL>((typename S::elem *)e.slope + row * a.N + col(u), a.N - col(u), d[u / 2]);
        }
      }
    });
  });
}

// ... -> the partial sums of a split contraction
template <int TI, int TJ>
__device__ __forceinline__ void la_partial(const Product &a, const la_f32x4 (&acc)[TI][TJ], int split, long long i, long long j) {
  la_each<TI * TJ / 2>([&](auto n_) __attribute__((always_inline)) {
    constexpr int t = decltype(n_)::value / (TJ / 2), u = decltype(n_)::value % (TJ / 2) * 2;
    const long long row = i + t * 16, c = j + u * 16, left = row < a.M ? a.N - c : 0;
    if (left <= 0) return;
    float y[8];
#pragma unroll
    for (int n = 0; n < 8; ++n) y[n] = acc[t][u + n / 4][n % 4];
    la_store8<HdF32, false>(a.partial + ((long long)split * a.M + row) * a.N + c, left, y);
  });
}

// workgroup `id` of a product's gi x gj tiles, part `split` of the contraction; ring: the LDS, 2 (BI + BJ) 128 bytes
template <class T, bool PROWS, bool QROWS, int WI, int WJ, int TI, int TJ, int ACT>
__device__ __forceinline__ void la_tile(const Product &a, int gi, int gj, int id, int split, char *ring) {
  constexpr int NT = 64 * WI * WJ, BI = WI * TI * 16, BJ = WJ * TJ * 16, KB = 8 * T::kPerVec, SLOT = (BI + BJ) * 128;
  typedef Operand<T, PROWS, false, BI, NT> OP;
  typedef Operand<T, QROWS, true, BJ, NT> OQ;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // workgroups go round robin over the 8 XCDs: give each XCD a contiguous run of tiles, walked in bands of 8 tile rows, so that the
  // operand panels of a band are shared in its L2
  int ti, tj;
  {
    const int n = gi * gj, per = n / 8, rem = n % 8, x = id % 8, q = id / 8;
    const int at = x * per + (x < rem ? x : rem) + q;
    const int band = at / (8 * gj), rows = gi - band * 8 < 8 ? gi - band * 8 : 8, in = at - band * 8 * gj;
    ti = band * 8 + in % rows;
    tj = in / rows;
  }
  const long long i0 = (long long)ti * BI, j0 = (long long)tj * BJ;
  const long long k0 = (long long)split * a.kchunk, k1 = k0 + a.kchunk < a.K ? k0 + a.kchunk : a.K;
  const int tiles = (int)((k1 - k0) / KB), rest = (int)((k1 - k0) % KB);
  const int wi = (wave % WI) * TI * 16, wj = (wave / WI) * TJ * 16;
  constexpr int L = OP::PER + OQ::PER;                 // direct loads per wave and tile
  OP op;
  OQ oq;
  op.init(a.p, a.ldp, i0, a.rp, k0, tid);
  oq.init(a.q, a.ldq, j0, a.rq, k0, tid);
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
  constexpr int GAP = TI * TJ * 3 / 4 / (TI + TJ) > 0 ? TI * TJ * 3 / 4 / (TI + TJ) : 1, LGAP = TI * TJ / L / 2 > 0 ? TI * TJ / L / 2 : 1;
  static_assert(TI + TJ <= TI * TJ && L <= TI * TJ, "room for the reads and the loads between the products");
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
    op.tail(ring, a.p, a.ldp, i0, a.rp, k0 + (long long)tiles * KB, k1, tid);
    oq.tail(ring + BI * 128, a.q, a.ldq, j0, a.rq, k0 + (long long)tiles * KB, k1, tid);
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
  if (a.splits > 1) la_partial(a, acc, split, i, j);
  else if (i0 + BI > a.M || j0 + BJ > a.N) {
    if (a.e.res) la_epilogue<T, ACT, false, true>(a, acc, i, j);
    else la_epilogue<T, ACT, false, false>(a, acc, i, j);
  } else {
    if (a.e.res) la_epilogue<T, ACT, true, true>(a, acc, i, j);
    else la_epilogue<T, ACT, true, false>(a, acc, i, j);
  }
}

template <class T, bool PROWS, bool QROWS, int WI, int WJ, int TI, int TJ, int ACT>
__global__ __launch_bounds__(64 * WI * WJ, 2) void la_tile_kernel(Product a, int gi, int gj) {
  __shared__ __align__(1024) char ring[2 * (WI * TI + WJ * TJ) * 16 * 128];
  const int id = (int)hd_block();
  if (id < gi * gj) la_tile<T, PROWS, QROWS, WI, WJ, TI, TJ, ACT>(a, gi, gj, id, blockIdx.z, ring);
}

// the split contraction joined in a fixed order, then the epilogue: four consecutive results per thread; the first `blocks`
// workgroups join x, the others w
template <class T>
__global__ __launch_bounds__(256) void la_join_kernel(Product x, Product w, unsigned blocks) {
  const Product &a = blockIdx.x < blocks ? x : w;
  const long long n = a.M * a.N, at = ((long long)(blockIdx.x < blocks ? blockIdx.x : blockIdx.x - blocks) * 256 + threadIdx.x) * 4;
  if (at >= n) return;
  float z[4] = {0.f, 0.f, 0.f, 0.f};
  if (at + 4 <= n) {
    for (int s = 0; s < a.splits; ++s) {
      float f[4];
      HdF32::unpack(hd_load16<HdF32>(a.partial + s * n + at), f);
#pragma unroll
      for (int q = 0; q < 4; ++q) z[q] += f[q];
    }
  } else {
    for (int s = 0; s < a.splits; ++s)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (at + q < n) z[q] += a.partial[s * n + at + q];
  }
  long long i = at / a.N, j = at - i * a.N;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    if (at + q < n) la_finish_any<T>(a.e, a.N, i, j, z[q]);
    if (++j == a.N) { j = 0; ++i; }
  }
}

// rows x cols at row stride ld -> rows at row stride `to` (a multiple of 16 bytes), the columns behind `cols` zero
struct Copy {
  long long rows, cols, ld, to;
  const void *src;
  void *dst;
};
// both operands of a product in one launch: the first `blocks` workgroups copy a, the others b
struct Copies {
  Copy a, b;
  unsigned blocks, all;
};
template <class T>
__device__ __forceinline__ void la_pad(const Copies &c_, unsigned id) {
  typedef typename T::elem elem;
  constexpr int VE = T::kPerVec;
  const Copy &o = id < c_.blocks ? c_.a : c_.b;
  const long long pieces = o.to / VE, at = (long long)(id < c_.blocks ? id : id - c_.blocks) * 256 + threadIdx.x;
  if (at >= o.rows * pieces) return;
  const long long r = at / pieces, c = (at - r * pieces) * VE;
  const elem *src = (const elem *)o.src + r * o.ld + c;
  float f[VE];
  if (c + VE <= o.cols) {
    hd_store16<T>((elem *)o.dst + r * o.to + c, hd_load16<T>(src));
  } else {
#pragma unroll
    for (int n = 0; n < VE; ++n) f[n] = c + n < o.cols ? T::load(src + n) : 0.f;
    hd_store16<T>((elem *)o.dst + r * o.to + c, T::pack(f));
  }
}

template <class T>
__global__ __launch_bounds__(256) void la_pad_kernel(Copies c) {
  la_pad<T>(c, (unsigned)hd_block());
}

// ----------------------------------------------------------------------------------------------------- the small kernels
// Few rows, or few results altogether: time is launches and round trips to memory, not products.  A workgroup owns (16 TI) x (16 TJ)
// results and its W waves split the contraction, step by step in turn; fragments go from global memory straight into registers, U
// steps in flight, with no LDS and no barrier before the one where the waves' sums are joined (in a fixed order) for the epilogue.
// DZ: P is dz, formed from dy and the slope as it is read, so that the whole backward pass of such a layer is one launch.
struct Small {
  Product a;
  const void *slope;        // DZ
  long long lds;            // its row stride
};

// the fragment values of row r at contraction indices k .. k + VE - 1 (the first `left` of them in range, others 0), as floats
template <class T, bool ROWS, bool FULL>
__device__ __forceinline__ void la_direct(const void *base, long long ld, long long r, long long k, long long left, float (&f)[T::kPerVec]) {
  const typename T::elem *p = (const typename T::elem *)base;
  if constexpr (!ROWS) {
    p += r * ld + k;
    if (FULL || left >= T::kPerVec) T::unpack(hd_load16<T>(p), f);
    else
#pragma unroll
      for (int n = 0; n < T::kPerVec; ++n) f[n] = n < left ? T::load(p + n) : 0.f;
  } else {
    p += k * ld + r;
#pragma unroll
    for (int n = 0; n < T::kPerVec; ++n) f[n] = FULL || n < left ? T::load(p + n * ld) : 0.f;
  }
}
template <class T, bool ROWS, bool FULL, bool DZ>
__device__ __forceinline__ hd_u32x4 la_direct_frag(const void *base, long long ld, const void *slope, long long lds, long long r,
                                                   long long k, long long left, float &sum) {
  if constexpr (!DZ && !ROWS) {
    if (FULL || left >= T::kPerVec) return hd_load16<T>((const typename T::elem *)base + r * ld + k);
  }
  float f[T::kPerVec];
  la_direct<T, ROWS, FULL>(base, ld, r, k, left, f);
  if constexpr (DZ) {
    if (slope) {
      float d[T::kPerVec];
      la_direct<typename SlopeOf<T>::type, ROWS, FULL>(slope, lds, r, k, left, d);
#pragma unroll
      for (int n = 0; n < T::kPerVec; ++n) f[n] *= d[n];
    }
    if constexpr (ROWS) {
#pragma unroll
      for (int n = 0; n < T::kPerVec; ++n) sum += f[n];
    }
  }
  return T::pack(f);
}

// db (DZ and ROWS only): the row sums of P are written there too (fp32 or T), by the workgroups of j0 = 0.  `lds`: 16 TI TJ W KB.
template <class T, bool PROWS, bool QROWS, int TI, int TJ, int W, bool DZ>
__device__ __forceinline__ void la_small_tile(const Small &s, long long i0, long long j0, void *db, int db_f32, float *lds) {
  constexpr int VE = T::kPerVec, KB = 4 * VE, NF = TI + TJ, U = PROWS || QROWS || DZ || NF > 4 ? 2 : 4;
  const Product &a = s.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 15, g = lane >> 4;
  long long pr[TI], qr[TJ];                            // rows out of range repeat the last one: never stored
#pragma unroll
  for (int t = 0; t < TI; ++t) pr[t] = i0 + t * 16 + r < a.M ? i0 + t * 16 + r : a.M - 1;
#pragma unroll
  for (int u = 0; u < TJ; ++u) qr[u] = j0 + u * 16 + r < a.N ? j0 + u * 16 + r : a.N - 1;
  la_f32x4 acc[TI][TJ] = {};
  float sum[TI];
#pragma unroll
  for (int t = 0; t < TI; ++t) sum[t] = 0.f;
  const bool sums = DZ && PROWS && db && j0 == 0;
  // Steps come in pairs (128 bytes of a K operand's rows: whole cache lines), wave w takes pairs w, w + W, ...; a group of U steps is
  // loaded while the one before is multiplied.
  constexpr int GK = U * W * KB;                       // contraction indices of a group, over all waves
  const long long groups = a.K / GK;
  constexpr int SETS = PROWS || QROWS ? 1 : 2;
  hd_u32x4 p[SETS][U][TI], q[SETS][U][TJ];
  auto load = [&](auto buf_, long long group) __attribute__((always_inline)) {
    constexpr int buf = decltype(buf_)::value;
#pragma unroll
    for (int n = 0; n < U; ++n) {
      const long long kk = group * GK + ((n / 2 * W + wave) * 2 + n % 2) * KB + g * VE;
#pragma unroll
      for (int t = 0; t < TI; ++t)
        p[buf][n][t] = la_direct_frag<T, PROWS, true, DZ>(a.p, a.ldp, s.slope, s.lds, pr[t], kk, VE, sum[t]);
#pragma unroll
      for (int u = 0; u < TJ; ++u) q[buf][n][u] = la_direct_frag<T, QROWS, true, false>(a.q, a.ldq, nullptr, 0, qr[u], kk, VE, sum[0]);
    }
    __builtin_amdgcn_sched_barrier(0);                 // all of them are on their way before the products below
  };
  auto multiply = [&](auto buf_) __attribute__((always_inline)) {
    constexpr int buf = decltype(buf_)::value;
#pragma unroll
    for (int n = 0; n < U; ++n)
#pragma unroll
      for (int t = 0; t < TI; ++t)
#pragma unroll
        for (int u = 0; u < TJ; ++u) acc[t][u] = la_mma(T{}, q[buf][n][u], p[buf][n][t], acc[t][u]);
    __builtin_amdgcn_sched_barrier(0);
  };
  if constexpr (PROWS || QROWS) {                      // (an R operand's loads are single elements: one set of registers is enough)
    for (long long m = 0; m < groups; ++m) {
      load(LaInt<0>{}, m);
      multiply(LaInt<0>{});
    }
  } else if (groups > 0) {
    load(LaInt<0>{}, 0);
    long long m = 0;
    for (; m + 2 < groups; m += 2) {
      load(LaInt<1>{}, m + 1);
      multiply(LaInt<0>{});
      load(LaInt<0>{}, m + 2);
      multiply(LaInt<1>{});
    }
    if (m + 1 < groups) {
      load(LaInt<1>{}, m + 1);
      multiply(LaInt<0>{});
      multiply(LaInt<1>{});
    } else {
      multiply(LaInt<0>{});
    }
  }
  long long k = groups * GK + (long long)wave * KB;
  for (; k < a.K; k += W * KB) {
    const long long kk = k + g * VE, left = a.K - kk;
    hd_u32x4 pt[TI], qt[TJ];
#pragma unroll
    for (int t = 0; t < TI; ++t)
      pt[t] = la_direct_frag<T, PROWS, false, DZ>(a.p, a.ldp, s.slope, s.lds, pr[t], kk, left, sum[t]);
#pragma unroll
    for (int u = 0; u < TJ; ++u) qt[u] = la_direct_frag<T, QROWS, false, false>(a.q, a.ldq, nullptr, 0, qr[u], kk, left, sum[0]);
#pragma unroll
    for (int t = 0; t < TI; ++t)
#pragma unroll
      for (int u = 0; u < TJ; ++u) acc[t][u] = la_mma(T{}, qt[u], pt[t], acc[t][u]);
  }
#pragma unroll
  for (int t = 0; t < TI; ++t)
#pragma unroll
    for (int u = 0; u < TJ; ++u) *reinterpret_cast<la_f32x4 *>(lds + ((wave * TI * TJ + t * TJ + u) * 64 + lane) * 4) = acc[t][u];
  __syncthreads();
  for (int e = tid; e < TI * TJ * 64; e += W * 64) {
    la_f32x4 z = *reinterpret_cast<const la_f32x4 *>(lds + e * 4);
#pragma unroll
    for (int w = 1; w < W; ++w) z += *reinterpret_cast<const la_f32x4 *>(lds + (w * TI * TJ * 64 + e) * 4);
    const int l = e & 63, tu = e >> 6;
    const long long i = i0 + (tu / TJ) * 16 + (l & 15), j = j0 + (tu % TJ) * 16 + (l >> 4) * 4;
    if (i >= a.M) continue;
#pragma unroll
    for (int n = 0; n < 4; ++n)
      if (j + n < a.N) la_finish_any<T>(a.e, a.N, i, j + n, z[n]);
  }
  if (sums) {                                          // uniform over the workgroup
    __syncthreads();
#pragma unroll
    for (int t = 0; t < TI; ++t) lds[(wave * TI + t) * 64 + lane] = sum[t];
    __syncthreads();
    for (int e = tid; e < TI * 16; e += W * 64) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w)
#pragma unroll
        for (int h = 0; h < 4; ++h) v += lds[(w * TI + e / 16) * 64 + h * 16 + e % 16];
      const long long i = i0 + e;
      if (i >= a.M) continue;
      if (db_f32) ((float *)db)[i] = v;
      else ((typename T::elem *)db)[i] = T::round(v);
    }
  }
}

template <class T, int TI, int TJ, int W>
__global__ __launch_bounds__(64 * W) void la_small_kernel(Product a) {
  __shared__ __align__(16) float lds[W * TI * TJ * 256];
  const long long gi = (a.M + 16 * TI - 1) / (16 * TI);
  const long long id = hd_block(), i0 = id % gi * (16 * TI), j0 = id / gi * (16 * TJ);
  if (j0 < a.N) la_small_tile<T, false, false, TI, TJ, W, false>(Small{a, nullptr, 0}, i0, j0, nullptr, 0, lds);
}

// dx and dW (and db) in one launch: the first `ndx` workgroups take tiles of dx, the others of dW
template <class T>
__global__ __launch_bounds__(256) void la_small_grad_kernel(Small x, Small w, int ndx, void *db, int db_f32) {
  __shared__ __align__(16) float lds[4 * 4 * 256];
  const int id = blockIdx.x;
  if (id < ndx) {
    const int gi = (int)((x.a.M + 31) / 32);
    la_small_tile<T, false, true, 2, 2, 4, true>(x, (long long)(id % gi) * 32, (long long)(id / gi) * 32, nullptr, 0, lds);
  } else {
    const int gi = (int)((w.a.M + 31) / 32), at = id - ndx;
    la_small_tile<T, true, true, 2, 2, 4, true>(w, (long long)(at % gi) * 32, (long long)(at / gi) * 32, db, db_f32, lds);
  }
}

// dz = dy slope (or dy, SLOPE false) at row stride ldz, or NULL, and column sums: a workgroup takes 64 x VE columns and a strip of rows, its four
// waves every fourth row; part (strips, N) fp32, or NULL.  Bound by its bytes (read dy and slope, write dz).  The workgroups behind
// those `blocks` make the padded copies that the products need.
template <class T, bool SLOPE>
__global__ __launch_bounds__(256) void la_dz_kernel(long long M, long long N, int strip, const void *dy_, long long ldy,
                                                    const void *slope_, void *dz_, long long ldz, float *part, unsigned blocks, Copies copies) {
  const unsigned id = (unsigned)hd_block();
  if (id >= blocks) {
    la_pad<T>(copies, id - blocks);
    return;
  }
  typedef typename T::elem elem;
  typedef typename SlopeOf<T>::type S;
  constexpr int VE = T::kPerVec, U = 4;
  __shared__ float sum[3][64][VE];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const unsigned across = (unsigned)((N + 64 * VE - 1) / (64 * VE)), down = id / across;
  const long long j = ((long long)(id - down * across) * 64 + lane) * VE, left = N - j;
  const long long i0 = (long long)down * strip, i1 = i0 + strip < M ? i0 + strip : M;
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
        }
        if (dz_) hd_store16<T>(dz + (i + 4 * u) * ldz, T::pack(f));
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
        }
        if (dz_) ((elem *)dz_)[i * ldz + j + n] = T::round(f);
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
      if (n < left) part[(long long)down * N + j + n] = (s[n] + sum[0][lane][n]) + (sum[1][lane][n] + sum[2][lane][n]);
  }
}

// the strips' sums joined: 64 columns per workgroup, its four waves every fourth strip
struct Sums {
  const float *part;
  long long N;
  int strips, db_f32;
  void *db;
};
template <class T>
__device__ __forceinline__ void la_db(const Sums &a, unsigned id, float (*sum)[64]) {
  constexpr int U = 16;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long long j = (long long)id * 64 + lane;
  float s = 0.f;
  if (j < a.N)
    for (int i = wave; i < a.strips; i += 4 * U) {     // a wave's round trips are what this costs: 128 strips each, 34 us one by one
      float f[U];
#pragma unroll
      for (int u = 0; u < U; ++u) f[u] = a.part[(long long)(i + 4 * u < a.strips ? i + 4 * u : i) * a.N + j];
#pragma unroll
      for (int u = 0; u < U; ++u) s += i + 4 * u < a.strips ? f[u] : 0.f;
    }
  if (wave) sum[wave - 1][lane] = s;
  __syncthreads();
  if (wave || j >= a.N) return;
  s = (s + sum[0][lane]) + (sum[1][lane] + sum[2][lane]);
  if (a.db_f32) ((float *)a.db)[j] = s;
  else ((typename T::elem *)a.db)[j] = T::round(s);
}
template <class T>
__global__ __launch_bounds__(256) void la_db_kernel(Sums a) {
  __shared__ float sum[3][64];
  la_db<T>(a, blockIdx.x, sum);
}

// dx, dW and db of a layer in the middle in one launch, on 64 x 64 tiles: `nx` workgroups for dx, `nw` for dW, the others for db.  Each
// of the products alone leaves the chip half idle and takes as long as its own loop: 1003 x 1001 -> 777 fp16 15 us for the three (36 one
// after the other), 2048 x 512 -> 512 bf16 forward and backward 28 us instead of 42.  Split contractions are joined by one more launch.
template <class T>
__global__ __launch_bounds__(256, 2) void la_pair_kernel(Product x, int xi, int xj, Product w, int wi, int wj, Sums b) {
  __shared__ __align__(1024) char ring[2 * 128 * 128];
  const int tx = xi * xj, tw = wi * wj, nx = tx * x.splits, nw = tw * w.splits, id = blockIdx.x;
  if (id < nx) la_tile<T, false, true, 2, 2, 2, 2, ACT_NONE>(x, xi, xj, id % tx, id / tx, ring);
  else if (id < nx + nw) la_tile<T, true, true, 2, 2, 2, 2, ACT_NONE>(w, wi, wj, (id - nx) % tw, (id - nx) / tw, ring);
  else la_db<T>(b, id - nx - nw, (float (*)[64])ring);
}

constexpr long long kMaxDim = 1LL << 31, kMaxStride = 1LL << 22;

inline long long la_div(long long a, long long b) { return (a + b - 1) / b; }
inline size_t la_align(size_t n) { return (n + 255) & ~(size_t)255; }
inline long long la_size(int dtype) { return dtype == PN2_DT_F32 ? 4 : 2; }
inline long long la_whole(long long n, int dtype) { return la_div(n, 16 / la_size(dtype)) * (16 / la_size(dtype)); }   // in 16-byte pieces

// Which kernel a product takes, and how often its contraction is split, by size and type.  Microseconds measured for bf16 unless
// said otherwise, this choice against the next one:
//   small   (no LDS, waves split the contraction) few rows, or few results: 1 x 4096 x 4096 8.2 against 16.8 for a split 64 x 64 tile,
//           72 x 512 x 256 4.1 against 7.9;  but 8 x 32768 x 2048 33 against 22, 32 x 8192 x 8192 46 against 27.  fp32, whose weights
//           cost twice: up to 16 rows always (16 x 8192 x 8192 61 against 74), and up to 512 x 512 (8.0 against 12.8)
//   64 x 64       up to 512 tiles: 1024^3 7.2 against 8.1 (128 x 64) and 11.0 (128 x 128)
//   128 x 64      2048^3 22.5 against 25.6 (64 x 64) and 24.5 (128 x 128);  fp32 128 against 127 and 134
//   128 x 128     fp32 from 512 such tiles on: 4096 x 4096 x 512 dW 147 against 167
//   256 x 256     16-bit, tiles for three quarters of the CUs: 8192^3 784 against 1248 (128 x 128)
// Splits only where a workgroup would walk a long contraction while CUs idle (a join costs a launch and the partial sums' traffic):
// 128 x 8192 x 8192 58 -> 35 with four, 64 x 4096 x 4096 21 -> 15 with four instead of two; 1024^3 7.2 -> 12.5 with two.
// Up to 64 fp32 tiles, whose products are slow, may split finer (forward and backward of 8192 x 64 -> 64 43 -> 32, 4096 x 512 -> 256 62
// -> 51); 16-bit ones would lose (8192 x 256 -> 256 31 -> 38).
enum { SMALL_11, SMALL_21, SMALL_22, TILE_64, TILE_128_64, TILE_128, TILE_256 };
struct Plan {
  int kernel, splits;
  long long kchunk;         // contraction indices per split
};

Plan la_plan(long long M, long long N, long long K, int dtype, bool small_ok) {
  const bool f32 = dtype == PN2_DT_F32;
  const long long n16 = la_div(M, 16) * la_div(N, 16);
  Plan p{TILE_64, 1, K};
  if (small_ok && K <= 16384) {
    if (M <= (f32 ? 16 : 4) || n16 <= 256) p.kernel = SMALL_11;
    else if (n16 <= 512 && (f32 || K <= 4096)) p.kernel = SMALL_21;
    else if ((f32 && n16 <= 1024) || (N <= 32 && K <= 1024)) p.kernel = SMALL_22;
    if (p.kernel != TILE_64) return p;
  }
  const long long t256 = la_div(M, 256) * la_div(N, 256), t128 = la_div(M, 128) * la_div(N, 128), t12864 = la_div(M, 128) * la_div(N, 64),
                  t64 = la_div(M, 64) * la_div(N, 64);
  long long tiles = t64;
  if (!f32 && t256 >= 192) { p.kernel = TILE_256; tiles = t256; }
  else if (f32 && t128 >= 512) { p.kernel = TILE_128; tiles = t128; }
  else if (t64 > 512) { p.kernel = TILE_128_64; tiles = t12864; }
  const long long kb = f32 ? 32 : 64, steps = la_div(K, kb);
  long long s = (p.kernel == TILE_256 ? 256 : 512) / tiles;
  const long long least = f32 && tiles > 64 ? 32 : f32 ? 8 : 16;      // tiles of 128 bytes a workgroup walks at least
  if (s > steps / least) s = steps / least;
  if (s < 1) s = 1;
  if (s > 64) s = 64;
  p.kchunk = la_div(steps, s) * kb;
  p.splits = (int)la_div(K, p.kchunk);
  return p;
}
size_t la_partial_bytes(const Plan &p, long long M, long long N) { return p.splits > 1 ? la_align((size_t)p.splits * M * N * 4) : 0; }

// An operand as it is, or as a padded copy: the tile kernels' direct loads need rows of whole 16-byte pieces at 16-byte addresses.
// rows x cols at row stride ld; an R operand's rows must also END with a piece.
struct Matrix {
  const void *p;
  long long rows, cols, ld;
  bool R;
};
bool la_direct_ok(const Matrix &o, int dtype) {
  return ((uintptr_t)o.p & 15) == 0 && o.ld * la_size(dtype) % 16 == 0 && o.ld <= kMaxStride && (!o.R || la_whole(o.cols, dtype) == o.cols);
}
size_t la_copy_bytes(const Matrix &o, int dtype) {
  return la_direct_ok(o, dtype) ? 0 : la_align((size_t)o.rows * la_whole(o.cols, dtype) * la_size(dtype));
}

struct Space {              // the caller's workspace, handed out piece by piece
  char *at;
  void *take(size_t n) {
    void *p = n ? at : nullptr;
    at += n;
    return p;
  }
};

// those of a and b that need it become padded copies (either may be NULL), which a kernel has yet to make
template <class T>
Copies la_copies(Matrix *a, Matrix *b, int dtype, Space &ws) {
  Copies c{};
  for (int n = 0; n < 2; ++n) {
    Matrix *o = n ? b : a;
    const size_t bytes = o ? la_copy_bytes(*o, dtype) : 0;
    if (bytes) {
      const long long to = la_whole(o->cols, dtype);
      (n ? c.b : c.a) = {o->rows, o->cols, o->ld, to, o->p, ws.take(bytes)};
      c.all += (unsigned)la_div(o->rows * (to / T::kPerVec), 256);
      o->p = (n ? c.b : c.a).dst;
      o->ld = to;
      if (o->R) o->cols = to;
    }
    if (!n) c.blocks = c.all;
  }
  return c;
}

inline unsigned la_joins(const Product &a) { return a.splits > 1 ? (unsigned)la_div(a.M * a.N, 1024) : 0; }

template <class T, bool PROWS, bool QROWS, int WI, int WJ, int TI, int TJ>
void la_tile_as(const Product &a, hipStream_t st) {
  const int gi = (int)la_div(a.M, WI * TI * 16), gj = (int)la_div(a.N, WJ * TJ * 16);
  constexpr int NT = 64 * WI * WJ;
  dim3 grid = hd_grid(gi * gj, NT);
  grid.z = (unsigned)a.splits;
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
  if (a.splits > 1) la_join_kernel<T><<<la_joins(a), 256, 0, st>>>(a, a, la_joins(a));
}

template <class T, int TI, int TJ, int W>
void la_small_as(const Product &a, hipStream_t st) {
  la_small_kernel<T, TI, TJ, W><<<hd_grid(la_div(a.M, 16 * TI) * la_div(a.N, 16 * TJ), 64 * W), 64 * W, 0, st>>>(a);
}

Product la_arguments(const Plan &plan, const Matrix &p, const Matrix &q, long long M, long long N, long long K, const Epilogue &e, Space ws) {
  Product a{};
  a.M = M; a.N = N; a.K = K;
  a.p = p.p; a.ldp = p.ld; a.rp = p.R ? p.cols : p.rows;
  a.q = q.p; a.ldq = q.ld; a.rq = q.R ? q.cols : q.rows;
  a.splits = plan.splits;
  a.kchunk = plan.kchunk;
  a.partial = (float *)ws.take(la_partial_bytes(plan, M, N));
  a.e = e;
  return a;
}

// C = P Q^T by the plan; P and Q are fit for it (padded where a tile kernel reads them)
template <class T, bool PROWS, bool QROWS>
int la_product(const Plan &plan, const Matrix &p, const Matrix &q, long long M, long long N, long long K, const Epilogue &e,
               Space ws, hipStream_t st) {
  const Product a = la_arguments(plan, p, q, M, N, K, e, ws);
  switch (plan.kernel) {
    case TILE_256:
      if constexpr (sizeof(typename T::elem) == 2) { la_tile_as<T, PROWS, QROWS, 2, 4, 8, 4>(a, st); break; }
      return PN2_EINVAL;                               // (never planned for fp32)
    case TILE_128:
      if constexpr (sizeof(typename T::elem) == 4) { la_tile_as<T, PROWS, QROWS, 2, 2, 4, 4>(a, st); break; }
      return PN2_EINVAL;                               // (never planned for 16-bit types)
    case TILE_128_64: la_tile_as<T, PROWS, QROWS, 2, 2, 4, 2>(a, st); break;
    case TILE_64: la_tile_as<T, PROWS, QROWS, 2, 2, 2, 2>(a, st); break;
    default:
      if constexpr (!PROWS && !QROWS) {
        if (plan.kernel == SMALL_11) la_small_as<T, 1, 1, 8>(a, st);
        else if (plan.kernel == SMALL_21) la_small_as<T, 2, 1, 8>(a, st);
        else la_small_as<T, 2, 2, 4>(a, st);
      }
  }
  return pn2_check_launch();
}

inline bool la_bad(long long M, long long N, long long K, int dtype) {
  return M < 0 || N < 1 || K < 1 || M >= kMaxDim || N > kMaxStride || K > kMaxStride || dtype < PN2_DT_F32 || dtype > PN2_DT_F16;
}

struct Forward {
  Plan plan;
  Matrix x, w;
  size_t bytes;
};
Forward la_forward_plan(long long M, long long N, long long K, int dtype, const void *x, long long ldx, const void *w, long long ldw) {
  Forward f;
  f.plan = la_plan(M, N, K, dtype, true);
  f.x = {x, M, K, ldx, false};
  f.w = {w, N, K, ldw, false};
  f.bytes = la_partial_bytes(f.plan, M, N);
  if (f.plan.kernel >= TILE_64) f.bytes += la_copy_bytes(f.x, dtype) + la_copy_bytes(f.w, dtype);
  return f;
}
template <class T>
int la_forward(Forward f, long long M, long long N, long long K, int dtype, const Epilogue &e, void *ws, hipStream_t st) {
  Space space{(char *)ws};
  if (f.plan.kernel >= TILE_64) {
    const Copies c = la_copies<T>(&f.x, &f.w, dtype, space);
    if (c.all) la_pad_kernel<T><<<hd_grid(c.all, 256), 256, 0, st>>>(c);
  }
  return la_product<T, false, false>(f.plan, f.x, f.w, M, N, K, e, space, st);
}

// rows per partial column sum: enough workgroups for the chip, at least 16 rows each, at most 512 strips
inline int la_strip(long long M, long long N, int dtype) {
  const long long cols = la_div(N, dtype == PN2_DT_F32 ? 256 : 512);
  long long strips = la_div(2048, cols);
  if (strips > 512) strips = 512;
  long long s = la_div(M, strips);
  return (int)(s < 16 ? 16 : s);
}

// The backward pass: one launch where everything is small (contractions of at most 4096); otherwise dz, db's strips and padded
// copies, then dx, dW and db: at once on 64 x 64 tiles, one after the other on larger ones.  Forward and backward in a graph, one launch
// against the others: fp32 up to 2^27 products (512^3 23 against 29 us, 1000 x 512 -> 256 31 against 42); 16-bit types, whose operands
// in row order the small kernel reads value by value, up to 2^24 (72 x 256 -> 512 13.6 against 13.3, and two launches fewer for the
// host; 512^3 18 against 16, 1000 x 512 -> 256 38 against 19) and 512 rows (512 x 64 -> 64 15.5 against 14.6, 2000 x 64 -> 64 50 against 22).
struct Backward {
  bool small, pair, own_dz;  // own_dz: dz is written (it is not dy itself)
  Plan px, pw;
  Matrix dz, dzr, w, x;   // dz as the K operand of dx and as the R operand of dW
  size_t dz_bytes, part, bytes;
};
Backward la_backward_plan(long long M, long long N, long long K, int dtype, const void *dy, long long ldy, bool slope, const void *x,
                          long long ldx, const void *w, long long ldw, int want) {
  Backward b{};
  b.small = (double)M * N * K <= (double)(1 << (dtype == PN2_DT_F32 ? 27 : 24)) && M <= (dtype == PN2_DT_F32 ? 2048 : 512) && N <= 4096 && (want & 3) && !((want & 4) && !(want & 2));
  if (b.small) return b;
  const bool products = (want & 3) != 0;
  b.dz = {dy, M, N, ldy, false};
  b.dzr = {dy, M, N, ldy, true};
  b.w = {w, N, K, ldw, true};
  b.x = {x, M, K, ldx, true};
  b.own_dz = products && (slope || !la_direct_ok(b.dz, dtype) || ((want & 2) && !la_direct_ok(b.dzr, dtype)));
  b.dz_bytes = b.own_dz ? la_align((size_t)M * la_whole(N, dtype) * la_size(dtype)) : 0;
  b.part = (want & 4) ? la_align((size_t)la_div(M, la_strip(M, N, dtype)) * N * 4) : 0;
  b.px = la_plan(M, K, N, dtype, false);
  b.pw = la_plan(N, K, M, dtype, false);
  b.pair = (want & 3) == 3 && b.px.kernel == TILE_64 && b.pw.kernel == TILE_64;
  const size_t copies = ((want & 1) ? la_copy_bytes(b.w, dtype) : 0) + ((want & 2) ? la_copy_bytes(b.x, dtype) : 0);
  // the two products use the rest one after the other, or at once
  const size_t dx = (want & 1) ? la_partial_bytes(b.px, M, K) : 0, dw = (want & 2) ? la_partial_bytes(b.pw, N, K) : 0;
  b.bytes = b.dz_bytes + b.part + copies + (b.pair ? dx + dw : dx > dw ? dx : dw);
  return b;
}

template <class T>
int la_backward(Backward b, long long M, long long N, long long K, int dtype, const void *dy, long long ldy, const void *slope,
                const void *x, long long ldx, const void *w, long long ldw, void *dx, void *dw, void *db, int db_f32, void *ws,
                hipStream_t st) {
  if (b.small) {
    Small sx{}, sw{};
    sx.a.M = M; sx.a.N = K; sx.a.K = N; sx.a.p = dy; sx.a.ldp = ldy; sx.a.q = w; sx.a.ldq = ldw; sx.a.e.y = dx; sx.slope = slope; sx.lds = N;
    sw.a.M = N; sw.a.N = K; sw.a.K = M; sw.a.p = dy; sw.a.ldp = ldy; sw.a.q = x; sw.a.ldq = ldx; sw.a.e.y = dw; sw.slope = slope; sw.lds = N;
    const long long ndx = dx ? la_div(M, 32) * la_div(K, 32) : 0, ndw = dw ? la_div(N, 32) * la_div(K, 32) : 0;
    la_small_grad_kernel<T><<<(unsigned)(ndx + ndw), 256, 0, st>>>(sx, sw, (int)ndx, db, db_f32);
    return pn2_check_launch();
  }
  Space space{(char *)ws};
  void *dz = space.take(b.dz_bytes);
  float *part = (float *)space.take(b.part);
  const long long ldz = la_whole(N, dtype);
  const Copies c = la_copies<T>(dx ? &b.w : nullptr, dw ? &b.x : nullptr, dtype, space);
  const int strip = la_strip(M, N, dtype);
  const Sums sums{part, N, (int)la_div(M, strip), db_f32, db};
  if (b.own_dz || db) {
    const unsigned blocks = (unsigned)(la_div(N, 64 * T::kPerVec) * sums.strips);
    const dim3 grid = hd_grid((long long)blocks + c.all, 256);
    if (slope) la_dz_kernel<T, true><<<grid, 256, 0, st>>>(M, N, strip, dy, ldy, slope, dz, ldz, part, blocks, c);
    else la_dz_kernel<T, false><<<grid, 256, 0, st>>>(M, N, strip, dy, ldy, nullptr, dz, ldz, part, blocks, c);
  } else if (c.all) {
    la_pad_kernel<T><<<hd_grid(c.all, 256), 256, 0, st>>>(c);
  }
  if (b.own_dz) {
    b.dz.p = b.dzr.p = dz;
    b.dz.ld = b.dzr.ld = b.dzr.cols = ldz;
  }
  const unsigned joins = db ? (unsigned)la_div(N, 64) : 0;
  Epilogue ex{}, ew{};
  ex.y = dx;
  ew.y = dw;
  if (b.pair) {
    const int xi = (int)la_div(M, 64), xj = (int)la_div(K, 64), wi = (int)la_div(N, 64);
    const Product px = la_arguments(b.px, b.dz, b.w, M, K, N, ex, space);
    space.take(la_partial_bytes(b.px, M, K));
    const Product pw = la_arguments(b.pw, b.dzr, b.x, N, K, M, ew, space);
    la_pair_kernel<T><<<(unsigned)(xi * xj * px.splits + wi * xj * pw.splits) + joins, 256, 0, st>>>(px, xi, xj, pw, wi, xj, sums);
    if (la_joins(px) + la_joins(pw)) la_join_kernel<T><<<la_joins(px) + la_joins(pw), 256, 0, st>>>(px, pw, la_joins(px));
    return pn2_check_launch();
  }
  if (db) la_db_kernel<T><<<joins, 256, 0, st>>>(sums);
  int rc = pn2_check_launch();
  if (rc == PN2_OK && dx) rc = la_product<T, false, true>(b.px, b.dz, b.w, M, K, N, ex, space, st);
  if (rc == PN2_OK && dw) rc = la_product<T, true, true>(b.pw, b.dzr, b.x, N, K, M, ew, space, st);
  return rc;
}

}  // namespace

extern "C" size_t pn2_linear_act_workspace_bytes(long long M, int N, int K, int dtype, const void *x, long long ldx, const void *w,
                                                 long long ldw) {
  if (la_bad(M, N, K, dtype) || M == 0) return 0;
  return la_forward_plan(M, N, K, dtype, x, ldx, w, ldw).bytes;
}

extern "C" int pn2_linear_act(long long M, int N, int K, int dtype, const void *x, long long ldx, const void *w, long long ldw,
                              const void *bias, int bias_dtype, int act, const void *residual, long long ldr, void *y, void *slope,
                              void *workspace, size_t workspace_bytes, void *stream) {
  if (la_bad(M, N, K, dtype) || act < ACT_NONE || act > ACT_SILU || ldx < 0 || ldw < 0 || ldr < 0 ||
      (bias && bias_dtype != dtype && bias_dtype != PN2_DT_F32))
    return PN2_EINVAL;
  if (M == 0) return PN2_OK;
  if (!x || !w || !y) return PN2_ENULL;
  const Forward f = la_forward_plan(M, N, K, dtype, x, ldx, w, ldw);
  if (workspace_bytes < f.bytes) return PN2_ENOSPC;
  if (f.bytes && !workspace) return PN2_ENULL;
  Epilogue e{};
  e.bias = bias; e.bias_f32 = bias_dtype == PN2_DT_F32; e.act = act; e.res = residual; e.ldr = ldr; e.y = y;
  e.slope = act == ACT_NONE ? nullptr : slope;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == PN2_DT_F32) return la_forward<HdF32>(f, M, N, K, dtype, e, workspace, st);
  if (dtype == PN2_DT_BF16) return la_forward<HdBF16>(f, M, N, K, dtype, e, workspace, st);
  return la_forward<HdF16>(f, M, N, K, dtype, e, workspace, st);
}

extern "C" size_t pn2_linear_act_grad_workspace_bytes(long long M, int N, int K, int dtype, const void *dy, long long ldy, int has_slope,
                                                      const void *x, long long ldx, const void *w, long long ldw, int want) {
  if (la_bad(M, N, K, dtype) || M == 0) return 0;
  return la_backward_plan(M, N, K, dtype, dy, ldy, has_slope != 0, x, ldx, w, ldw, want).bytes;
}

extern "C" int pn2_linear_act_grad(long long M, int N, int K, int dtype, const void *dy, long long ldy, const void *slope,
                                   const void *x, long long ldx, const void *w, long long ldw, void *dx, void *dw, void *db,
                                   int db_dtype, void *workspace, size_t workspace_bytes, void *stream) {
  if (la_bad(M, N, K, dtype) || M < 1 || ldy < 0 || ldx < 0 || ldw < 0 || (db && db_dtype != dtype && db_dtype != PN2_DT_F32))
    return PN2_EINVAL;
  if (!dy || (dx && !w) || (dw && !x)) return PN2_ENULL;
  const int want = (dx ? 1 : 0) | (dw ? 2 : 0) | (db ? 4 : 0);
  if (!want) return PN2_OK;
  const Backward b = la_backward_plan(M, N, K, dtype, dy, ldy, slope != nullptr, x, ldx, w, ldw, want);
  if (workspace_bytes < b.bytes) return PN2_ENOSPC;
  if (b.bytes && !workspace) return PN2_ENULL;
  hipStream_t st = (hipStream_t)stream;
  const int f32 = db_dtype == PN2_DT_F32;
  if (dtype == PN2_DT_F32) return la_backward<HdF32>(b, M, N, K, dtype, dy, ldy, slope, x, ldx, w, ldw, dx, dw, db, f32, workspace, st);
  if (dtype == PN2_DT_BF16) return la_backward<HdBF16>(b, M, N, K, dtype, dy, ldy, slope, x, ldx, w, ldw, dx, dw, db, f32, workspace, st);
  return la_backward<HdF16>(b, M, N, K, dtype, dy, ldy, slope, x, ldx, w, ldw, dx, dw, db, f32, workspace, st);
}
