// head_common.h — element types, wave reductions and 16-byte vectors shared by the dense-head kernels (label_probs.hip,
// linear_act.hip).
#pragma once
#include "pn2_common.h"

namespace {

typedef unsigned hd_u32x4 __attribute__((ext_vector_type(4)));
// 16 bytes at any element boundary: rows of an odd length start anywhere, and gfx950 loads and stores dwordx4 unaligned
// (may_alias: the same memory is also accessed as elements)
typedef unsigned hd_u32x4_any __attribute__((ext_vector_type(4), aligned(2), may_alias));
typedef __bf16 hd_bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 hd_f16x2 __attribute__((ext_vector_type(2)));
typedef float hd_f32x2 __attribute__((ext_vector_type(2)));

// element types: kPerVec values per 16 bytes, unpack to float, pack with round to nearest even
struct HdF32 {
  typedef float elem;
  static constexpr int kPerVec = 4;
  static __device__ __forceinline__ float load(const elem *p) { return *p; }
  static __device__ __forceinline__ elem round(float v) { return v; }
  static __device__ __forceinline__ void unpack(hd_u32x4 w, float (&f)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned u = w[i];                         // (a bit_cast of the vector's element itself reads element 0)
      f[i] = __builtin_bit_cast(float, u);
    }
  }
  static __device__ __forceinline__ hd_u32x4 pack(const float (&f)[4]) {
    hd_u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __builtin_bit_cast(unsigned, f[i]);
    return w;
  }
};

struct HdBF16 {
  typedef __bf16 elem;
  static constexpr int kPerVec = 8;
  static __device__ __forceinline__ float load(const elem *p) { return (float)*p; }
  static __device__ __forceinline__ elem round(float v) { return (elem)v; }
  static __device__ __forceinline__ void unpack(hd_u32x4 w, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned u = w[i];
      f[2 * i] = __builtin_bit_cast(float, u << 16);
      f[2 * i + 1] = __builtin_bit_cast(float, u & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ unsigned pack2(float a, float b) {
    return __builtin_bit_cast(unsigned, __builtin_convertvector(hd_f32x2{a, b}, hd_bf16x2));
  }
  static __device__ __forceinline__ hd_u32x4 pack(const float (&f)[8]) {
    return hd_u32x4{pack2(f[0], f[1]), pack2(f[2], f[3]), pack2(f[4], f[5]), pack2(f[6], f[7])};
  }
};

struct HdF16 {
  typedef _Float16 elem;
  static constexpr int kPerVec = 8;
  static __device__ __forceinline__ float load(const elem *p) { return (float)*p; }
  static __device__ __forceinline__ elem round(float v) { return (elem)v; }
  static __device__ __forceinline__ void unpack(hd_u32x4 w, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned u = w[i];
      const hd_f16x2 h = __builtin_bit_cast(hd_f16x2, u);
      f[2 * i] = (float)h.x;
      f[2 * i + 1] = (float)h.y;
    }
  }
  static __device__ __forceinline__ unsigned pack2(float a, float b) {
    return __builtin_bit_cast(unsigned, __builtin_convertvector(hd_f32x2{a, b}, hd_f16x2));
  }
  static __device__ __forceinline__ hd_u32x4 pack(const float (&f)[8]) {
    return hd_u32x4{pack2(f[0], f[1]), pack2(f[2], f[3]), pack2(f[4], f[5]), pack2(f[6], f[7])};
  }
};

template <class T>
__device__ __forceinline__ hd_u32x4 hd_load16(const typename T::elem *p) {
  return *reinterpret_cast<const hd_u32x4_any *>(p);
}
template <class T>
__device__ __forceinline__ void hd_store16(typename T::elem *p, hd_u32x4 w) {
  *reinterpret_cast<hd_u32x4_any *>(p) = w;
}

template <int CTRL>
__device__ __forceinline__ float hd_dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, false));
}

// Wave-wide sum / maximum in a fixed order (DPP inside the rows of 16, then the four rows); the result is wave-uniform.
__device__ __forceinline__ float hd_wave_sum(float v) {
  v += hd_dpp<PN2_DPP_QUAD_XOR1>(v);
  v += hd_dpp<PN2_DPP_QUAD_XOR2>(v);
  v += hd_dpp<PN2_DPP_ROW_HALF_MIRROR>(v);
  v += hd_dpp<PN2_DPP_ROW_MIRROR>(v);
  return (pn2_readlane_f32(v, 0) + pn2_readlane_f32(v, 16)) + (pn2_readlane_f32(v, 32) + pn2_readlane_f32(v, 48));
}
__device__ __forceinline__ float hd_wave_max(float v) {
  v = fmaxf(v, hd_dpp<PN2_DPP_QUAD_XOR1>(v));
  v = fmaxf(v, hd_dpp<PN2_DPP_QUAD_XOR2>(v));
  v = fmaxf(v, hd_dpp<PN2_DPP_ROW_HALF_MIRROR>(v));
  v = fmaxf(v, hd_dpp<PN2_DPP_ROW_MIRROR>(v));
  return fmaxf(fmaxf(pn2_readlane_f32(v, 0), pn2_readlane_f32(v, 16)), fmaxf(pn2_readlane_f32(v, 32), pn2_readlane_f32(v, 48)));
}

__device__ __forceinline__ float hd_exp2(float v) { return __builtin_amdgcn_exp2f(v); }   // v_exp_f32: 1 ulp, flushes below 2^-126

// n workgroups of `threads` threads.  The launch packet counts an axis in 32-bit threads, and 2^32 of them wrap without an error (67
// million short rows got 4 of their results): what passes that goes to the second axis.  hd_block(): this workgroup's number, which
// can then be n or more.
inline dim3 hd_grid(long long n, unsigned threads) {
  const long long most = 0xffffffffLL / threads, y = (n + most - 1) / most;
  return y > 1 ? dim3((unsigned)((n + y - 1) / y), (unsigned)y) : dim3((unsigned)n);
}
__device__ __forceinline__ long long hd_block() { return (long long)blockIdx.y * gridDim.x + blockIdx.x; }

constexpr float kHdInf = __builtin_huge_valf();
constexpr float kHdLog2e = 1.4426950408889634f;
constexpr float kHdLn2 = 0.6931471805599453f;

}  // namespace
