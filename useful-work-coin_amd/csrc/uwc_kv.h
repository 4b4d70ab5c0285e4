// Shared pieces of the paged 8-bit key/value cache's kernels (uwc_kv_cache.hip, uwc_kv_attend.hip).
//
// One layer's cache: keys int8 (pages, Hkv, P, hd), values int8 (pages, Hkv, hd, P) with the tokens
// innermost, fp32 scales (pages, Hkv) of either; token p of sequence b lies in slot p % P of page
// table[b][p / P]. P is 16, 32, 64 or 128, so 16 consecutive tokens from a multiple of 16 (a granule)
// always share a page and its scale. The offset of a page is held in 64 bits.
//
// Whatever device-side numbers say (table entries, lengths, cu), no kernel leaves the buffers: a page
// that is needed but outside [0, pages) makes the rows that need it NaN, and rows outside [0, T) are
// not touched.
#pragma once
#include "uwc_common.h"

#define KV_AI __attribute__((always_inline))

typedef _Float16 h2v __attribute__((ext_vector_type(2)));
typedef _Float16 h4v __attribute__((ext_vector_type(4)));
typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef __bf16 b8v __attribute__((ext_vector_type(8)));
typedef u32 u4v __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));

template <class T>
struct kv_vec;
template <>
struct kv_vec<_Float16> {
  typedef h8v v8;
};
template <>
struct kv_vec<__bf16> {
  typedef b8v v8;
};

// The packed rows of the call: sequence b's new tokens are rows cu[b] .. cu[b + 1] - 1 (cu NULL: one each).
struct KvRows {
  const int* cu;
  int B, T;
};

__device__ __forceinline__ int kv_new(const KvRows& R, int b) {
  if (!R.cu) return 1;
  const int n = R.cu[b + 1] - R.cu[b];
  return n < 0 ? 0 : n > R.T ? R.T : n;
}

// Finds unit number `unit` of the list in which sequence b has count(b) units: its sequence and its index
// there, the same in every lane of the wave. False past the list's end; unit then holds its distance from it.
template <class F>
__device__ __forceinline__ bool kv_find(int& unit, int B, F&& count, int& b, int& j) {
  const int lane = threadIdx.x & 63;
  for (int base = 0; base < B; base += 64) {
    const int n = base + lane < B ? count(base + lane) : 0;
    int s = n;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int up = __shfl_up(s, d, 64);
      if (lane >= d) s += up;
    }
    const int total = __shfl(s, 63, 64);
    if (unit < total) {
      const int l = __builtin_ctzll(__ballot(s > unit));
      b = __builtin_amdgcn_readfirstlane(base + l);
      j = __builtin_amdgcn_readfirstlane(unit - (__shfl(s, l, 64) - __shfl(n, l, 64)));
      return true;
    }
    unit -= total;
  }
  unit = __builtin_amdgcn_readfirstlane(unit);
  return false;
}

__device__ __forceinline__ u32 kv_umax_wave(u32 v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    const u32 o = (u32)__shfl_xor((int)v, d, 64);
    v = o > v ? o : v;
  }
  return v;
}

__device__ __forceinline__ float kv_nan() { return __uint_as_float(0x7fc00000u); }
