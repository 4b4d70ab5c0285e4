// Shared pieces of the kernels with 4-bit weights (uwc_w4.hip, uwc_w4_gemm.hip).
//
//   y[m, n] = sum_k x[m, k] w[n, k],   w[n, k] = value(code[n, k]) 2^(scale[n, k / 32] - 127)
//
// with value(code) = 0, 0.5, 1, 1.5, 2, 3, 4, 6 and the same negated: the fp4 elements and power-of-two group scales
// of the OCP microscaling format. A row's codes are K / 2 bytes, the weight of the lower k in a byte's low half;
// its scales K / 32 bytes. value times a power of two is exact in bf16 (two bits of 8), so the matrix instructions take the
// true weights, as long as those are below 2^128 (any of scales up to 252; larger ones are infinite). fp16 has less range: weights of float16
// rows are rounded to it (exact for scales from 104 to 140; 65520 and more is infinite).
#pragma once
#include "uwc_common.h"

#define W4_AI __attribute__((always_inline))

typedef _Float16 w4_h2 __attribute__((ext_vector_type(2)));
typedef _Float16 w4_h8 __attribute__((ext_vector_type(8)));
typedef __bf16 w4_b2 __attribute__((ext_vector_type(2)));
typedef __bf16 w4_b8 __attribute__((ext_vector_type(8)));
typedef u32 w4_u4 __attribute__((ext_vector_type(4)));
typedef float w4_f16 __attribute__((ext_vector_type(16)));

template <class T>
struct W4;
template <>
struct W4<__bf16> {
  typedef w4_b8 v8;
  // the weights of a dword's eight codes: one instruction for a byte's two and their scale, whose exponent alone counts
  static __device__ __forceinline__ v8 weights(u32 codes, float scale) {
    const w4_b2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1),
                c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3);
    return v8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
  }
  static __device__ __forceinline__ f4v mul(v8 a, v8 b, f4v c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ w4_f16 mul32(v8 a, v8 b, w4_f16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct W4<_Float16> {
  typedef w4_h8 v8;
  static __device__ __forceinline__ v8 weights(u32 codes, float scale) {
    const w4_h2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 1),
                c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 3);
    return v8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
  }
  static __device__ __forceinline__ f4v mul(v8 a, v8 b, f4v c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ w4_f16 mul32(v8 a, v8 b, w4_f16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};

// The call: rows of x are x_stride elements apart, those of y dense. F: outputs of a row. The weight has N rows; where
// `gated`, N = 2 F, and output f comes of rows f and F + f.
struct W4Args {
  const void* x;
  long x_stride;
  const u8 *codes, *scales;
  const void* bias;
  void* y;
  int M, F, N, K;
};

__device__ __forceinline__ float w4_silu(float g) { return g / (1.0f + __expf(-g)); }

// v + bias for outputs n .. n + 3
template <class T>
__device__ __forceinline__ f4v w4_bias(const W4Args& a, int n, f4v v) {
  if (a.bias) {
    const T* b = static_cast<const T*>(a.bias);
#pragma unroll
    for (int r = 0; r < 4; r++) v[r] += (float)b[n + r < a.F ? n + r : a.F - 1];
  }
  return v;
}

// Four outputs n .. n + 3 of row m; four at once where rows of y stay aligned to that.
template <class T>
__device__ __forceinline__ void w4_store(const W4Args& a, int m, int n, f4v v) {
  typedef T v4 __attribute__((ext_vector_type(4)));
  T* y = static_cast<T*>(a.y) + (long)m * a.F + n;
  v = w4_bias<T>(a, n, v);
  if (a.F % 4 == 0) {
    v4 o = {(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
    *reinterpret_cast<v4*>(y) = o;
  } else {
#pragma unroll
    for (int r = 0; r < 4; r++)
      if (n + r < a.F) y[r] = (T)v[r];
  }
}

// The kernel for many rows (uwc_w4_gemm.hip), and about how many us it takes.
float w4_gemm_us(const W4Args& a, bool gated);
int w4_gemm(const char* fn, const W4Args& a, int dtype, bool gated, hipStream_t stream);
