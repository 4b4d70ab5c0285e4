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

// A unit of work: number j of sequence b's, whose new rows are row0 .. row0 + n - 1, and its entry x of the call's
// per-sequence numbers (tokens cached before, or after).
struct KvUnit {
  int b, j, row0, n, x;
};

// Finds unit number `unit` of the list in which a sequence of n new rows and number x has count(n, x) units, uniform over
// the wave as `unit` has to be. False past the list's end; unit then holds its distance from it. A sequence's numbers are
// loaded once, by the lane that counts its units. For packed rows (R.cu).
template <class F>
__device__ __forceinline__ bool kv_find(const KvRows& R, const int* xs, int& unit, F&& count, KvUnit& u) {
  const int lane = threadIdx.x & 63;
  int c0 = 0, x = 0, n = 0;
  auto load = [&](int i) KV_AI {
    if (i >= R.B) return c0 = x = n = 0, 0;
    c0 = R.cu[i], x = xs[i], n = R.cu[i + 1] - c0;
    n = n < 0 ? 0 : n > R.T ? R.T : n;
    return count(n, x);
  };
  for (int base = 0; base < R.B; base += 64) {
    const int units = load(base + lane);
    // the inclusive sums over the lanes: within rows of 16, then of the rows before
    int s = units;
    s += __builtin_amdgcn_update_dpp(0, s, 0x111, 0xf, 0xf, true);  // row_shr:1, :2, :4, :8
    s += __builtin_amdgcn_update_dpp(0, s, 0x112, 0xf, 0xf, true);
    s += __builtin_amdgcn_update_dpp(0, s, 0x114, 0xf, 0xf, true);
    s += __builtin_amdgcn_update_dpp(0, s, 0x118, 0xf, 0xf, true);
    s += __builtin_amdgcn_update_dpp(0, s, 0x142, 0xa, 0xf, false);  // row_bcast:15 into rows 1 and 3
    s += __builtin_amdgcn_update_dpp(0, s, 0x143, 0xc, 0xf, false);  // row_bcast:31 into rows 2 and 3
    const int total = __builtin_amdgcn_readlane(s, 63);
    if (unit < total) {
      const int l = __builtin_ctzll(__ballot(s > unit));
      u.b = base + l;
      u.j = unit - (__builtin_amdgcn_readlane(s, l) - __builtin_amdgcn_readlane(units, l));
      u.row0 = __builtin_amdgcn_readlane(c0, l), u.n = __builtin_amdgcn_readlane(n, l), u.x = __builtin_amdgcn_readlane(x, l);
      return true;
    }
    unit -= total;
  }
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
