// Linears with 4-bit weights for few rows: the weights are streamed once per 16 or 32 rows, straight from memory into
// the registers that the matrix instructions read.
//
// Bytes bound it, or at few of them a launch and the latency of its loads: one row of 2 x 14336 x 4096, gated, 17.3 us (62 MB, 3.6 TB/s;
// 10.2 at the rate of a streaming read), one of 2048 x 2048 3.7 us.
#include "uwc_w4.h"

namespace {

// A workgroup makes 16 NT weight rows times 16 MT rows of x (where GATED, 8 NT outputs: half of the NT tiles are gate
// rows, half the matching up rows); its waves take every W-th unit of 256 k and add up in LDS. In a unit, lane
// (i = lane % 16, j = lane / 16) holds weight row i's groups 2 j and 2 j + 1, 64 codes in 32 bytes with two scales, and x row i's
// same 64 values; step t multiplies elements 8 t .. 8 t + 7 of the first groups, step 4 + t of the second, so the k order inside
// a unit differs from memory's, alike for both. Whole lines of 128 bytes of codes are read, and all of a wave's first two units at once.
template <class T, int MT, int NT, int W, bool GATED>
__global__ __launch_bounds__(64 * W) void w4_rows_kernel(W4Args a, int nb, int mb) {
  typedef typename W4<T>::v8 v8;
  constexpr int OT = GATED ? NT / 2 : NT;  // tiles of outputs
  __shared__ f4v red[W * MT * NT * 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // the workgroups of one weight block on one XCD: its L2 then reads the weights once
  const int id = blockIdx.x, n_blk = id / (8 * mb) * 8 + id % 8, m_blk = id / 8 % mb;
  if (n_blk >= nb) return;
  const int i = lane & 15, j = lane >> 4, groups = a.K / 32, units = (groups + 7) / 8;
  const int n0 = n_blk * 16 * OT, m0 = m_blk * 16 * MT;
  const u8 *cp[NT], *sp[NT];
#pragma unroll
  for (int t = 0; t < NT; t++) {
    int n = n0 + 16 * (t % OT) + i;
    n = (n < a.F ? n : a.F - 1) + (t >= OT ? a.F : 0);  // rows past the last are read twice and not stored
    cp[t] = a.codes + (long)n * (a.K / 2);
    sp[t] = a.scales + (long)n * groups;
  }
  const T* xp[MT];
  bool there[MT];
#pragma unroll
  for (int t = 0; t < MT; t++) {
    const int m = m0 + 16 * t + i;
    there[t] = m < a.M;
    xp[t] = static_cast<const T*>(a.x) + (long)(there[t] ? m : 0) * a.x_stride;
  }
  f4v acc[MT][NT];
#pragma unroll
  for (int p = 0; p < MT; p++)
#pragma unroll
    for (int t = 0; t < NT; t++) acc[p][t] = f4v{0, 0, 0, 0};

  struct Weights {
    w4_u4 c[NT][2];
    u32 s[NT];
  };
  struct Rows {
    v8 x[MT][8];
  };
  auto load = [&](Weights& p, int u) W4_AI {
    // groups that are not there are others of the row, which meet zeros of x
    const int g = 8 * u + 2 * j, g0 = g < groups ? g : groups - 1, g1 = g + 1 < groups ? g + 1 : groups - 1;
    const int pair = g0 < groups - 1 ? g0 : groups - 2;
#pragma unroll
    for (int t = 0; t < NT; t++) {
      p.c[t][0] = *reinterpret_cast<const w4_u4*>(cp[t] + g0 * 16);
      p.c[t][1] = *reinterpret_cast<const w4_u4*>(cp[t] + g1 * 16);
      if (groups > 1) {
        unsigned short two;  // at any address: rows may hold an odd number of scales
        __builtin_memcpy(&two, sp[t] + pair, 2);
        p.s[t] = (u32)two >> (8 * (g0 - pair));
      } else {
        p.s[t] = *sp[t];
      }
    }
  };
  auto load_rows = [&](Rows& p, int u) W4_AI {
    const int g = 8 * u + 2 * j;
#pragma unroll
    for (int q = 0; q < MT; q++)
#pragma unroll
      for (int t = 0; t < 8; t++) {
        v8 z = {};
        if (there[q] && g + t / 4 < groups) z = *reinterpret_cast<const v8*>(xp[q] + g * 32 + t * 8);
        p.x[q][t] = z;
      }
  };
  auto mul = [&](const Weights& p, const Rows& r) W4_AI {
#pragma unroll
    for (int t = 0; t < 8; t++)
#pragma unroll
      for (int n = 0; n < NT; n++) {
        const v8 w = W4<T>::weights(p.c[n][t / 4][t % 4], __uint_as_float((p.s[n] >> (t / 4 * 8) & 0xff) << 23));
#pragma unroll
        for (int q = 0; q < MT; q++) acc[q][n] = W4<T>::mul(w, r.x[q][t], acc[q][n]);
      }
  };
  // the next unit's weights are on their way while this one is multiplied; its x too where one tile a wave leaves registers for that
  int u = wave;
  if (u < units) {
    Weights now;
    Rows x;
    load(now, u);
    load_rows(x, u);
    for (; u + W < units; u += W) {
      Weights next;
      load(next, u + W);
      if constexpr (MT == 1 && NT == 1) {
        Rows nx;
        load_rows(nx, u + W);
        mul(now, x);
        x = nx;
      } else {
        mul(now, x);
        load_rows(x, u + W);
      }
      now = next;
    }
    mul(now, x);
  }
  // lane (i, j) holds outputs 4 j .. 4 j + 3 of row i; sums over the waves in their order
#pragma unroll
  for (int q = 0; q < MT; q++)
#pragma unroll
    for (int t = 0; t < NT; t++) red[((wave * MT + q) * NT + t) * 64 + lane] = acc[q][t];
  __syncthreads();
  for (int e = threadIdx.x; e < MT * OT * 64; e += 64 * W) {
    const int q = e / (OT * 64), t = e / 64 % OT, l = e % 64;
    auto sum = [&](int t) W4_AI {
      f4v v = red[(q * NT + t) * 64 + l];
      for (int w = 1; w < W; w++) v += red[((w * MT + q) * NT + t) * 64 + l];
      return v;
    };
    f4v v = sum(t);
    if (GATED) {
      const f4v u = sum(OT + t);
#pragma unroll
      for (int r = 0; r < 4; r++) v[r] = w4_silu(v[r]) * u[r];
    }
    const int m = m0 + 16 * q + (l & 15), n = n0 + 16 * t + 4 * (l >> 4);
    if (m < a.M && n < a.F) w4_store<T>(a, m, n, v);
  }
}

template <class T, int MT, int NT, int W, bool GATED>
int rows(const char* fn, const W4Args& a, hipStream_t stream) {
  constexpr int out = 16 * (GATED ? NT / 2 : NT);
  const long nb = ((long)a.F + out - 1) / out, mb = ((long)a.M + 16 * MT - 1) / (16 * MT);
  const long blocks = (nb + 7) / 8 * 8 * mb;
  if (blocks > 0xFFFFFFFFL / (64 * W)) return uwc_fail("%s: too many rows (%d) and outputs (%d)", fn, a.M, a.F);
  hipLaunchKernelGGL((w4_rows_kernel<T, MT, NT, W, GATED>), dim3((unsigned)blocks), dim3(64 * W), 0, stream, a, (int)nb, (int)mb);
  return uwc_launch_status(fn);
}

// About how many us the kernel above takes past 16 rows: the eight waves of a workgroup take a unit each at a time, which lasts `one` us or, where
// the workgroups wait for each other's loads, one for every `many` of them.
// Against the tiles in LDS, K = 14016: 69 x 500 17 us (41 there), 128 x 1024 40 (43), 333 x 500 65 (45); K = 2048: 24 x 1024 5.0 (9.8),
// 333 x 500 10.6 (10.0), 333 x 1024 18 (10).
float few_rows_us(const W4Args& a, int tiles_of_x, float one, float many) {
  const long units = (a.K + 255) / 256, groups = ((long)a.M + 16 * tiles_of_x - 1) / (16 * tiles_of_x) * (((long)a.F + 15) / 16);
  const float each = groups / many;
  return 2.9f + (units + 7) / 8 * (each > one ? each : one);
}

// More tiles of weights to a workgroup share the loads of x, which take longer than the codes from about four rows on (64 lines of
// memory an instruction against 16); fewer, and more waves to a tile, keep all compute units at work. us, weights from HBM:
//   gated, tiles x waves    2 x 4   4 x 4   2 x 8        linear                  1 x 8   2 x 8   4 x 4
//   1 x 14336 x 4096         18.2    19.4    19.8        1 x 4096 x 14336         13.2    19.4    50.2
//   16 x 14336 x 4096        40.1    25.2    39.9        13 x 6144 x 4096         12.3     8.9    12.8
//   1 x 6144 x 2048           6.5     7.6     6.8        8 x 28672 x 4096         32.1    25.5    20.5
//   1 x 2048 x 8192          14.6             10.3       (16 waves to a tile: within 3% of 8, 1 x 4096 x 14336 12.6)
//   1 x 203 x 11104          17.0             11.2
//   16 x 4096 x 4096                  15.3    11.5
//   16 x 6144 x 4096                  15.7    19.3
template <class T>
int run(const char* fn, const W4Args& a, bool gated, hipStream_t stream) {
  if (gated) {
    if (a.M > 16 || a.F <= 4608) return rows<T, 1, 2, 8, true>(fn, a, stream);
    return a.M > 4 ? rows<T, 1, 4, 4, true>(fn, a, stream) : rows<T, 1, 2, 4, true>(fn, a, stream);
  }
  if (a.M <= 16) {
    if (a.F >= 16384) return rows<T, 1, 4, 4, false>(fn, a, stream);
    if (a.F >= 6144) return rows<T, 1, 2, 8, false>(fn, a, stream);
    return rows<T, 1, 1, 8, false>(fn, a, stream);
  }
  return few_rows_us(a, 1, 2, 85) <= few_rows_us(a, 2, 3.2f, 50) ? rows<T, 1, 1, 8, false>(fn, a, stream) : rows<T, 2, 1, 8, false>(fn, a, stream);
}

int call(const char* fn, const W4Args& a, int dtype, bool gated, hipStream_t stream) {
  if (dtype != UWC_W4_BF16 && dtype != UWC_W4_FP16) return uwc_fail("%s: unknown dtype %d", fn, dtype);
  if (a.M < 0 || a.F < 0 || (gated && a.F > 0x3fffffff)) return uwc_fail("%s: bad M=%d N=%d", fn, a.M, a.F);
  if (a.K <= 0 || a.K % 32 || a.K > 1 << 22) return uwc_fail("%s: K=%d must be a positive multiple of 32, at most 2^22", fn, a.K);
  if (a.M == 0 || a.F == 0) return UWC_OK;
  if (!a.x || !a.codes || !a.scales || !a.y) return uwc_fail("%s: null arguments", fn);
  if (a.x_stride > 1 << 22) return uwc_fail("%s: rows of x are %ld elements apart, more than 2^22", fn, a.x_stride);
  if (a.x_stride < 0 || a.x_stride % 8 || (((uintptr_t)a.x | (uintptr_t)a.codes) & 15) || ((uintptr_t)a.y & 7))
    return uwc_fail("%s: rows of x and codes must be 16-byte aligned, y 8-byte aligned", fn);
  if (a.M > 16) {
    const float one = few_rows_us(a, 1, gated ? 3 : 2, gated ? 75 : 85), two = gated ? one : few_rows_us(a, 2, 3.2f, 50);
    if (w4_gemm_us(a, gated) < (one < two ? one : two)) return w4_gemm(fn, a, dtype, gated, stream);
  }
  return dtype == UWC_W4_BF16 ? run<__bf16>(fn, a, gated, stream) : run<_Float16>(fn, a, gated, stream);
}

}  // namespace

extern "C" int uwc_w4_linear(const void* x, int64_t x_stride, int dtype, int M, const uint8_t* codes, const uint8_t* scales,
                             int N, int K, const void* bias, void* y, hipStream_t stream) {
  return call("uwc_w4_linear", W4Args{x, (long)x_stride, codes, scales, bias, y, M, N, N, K}, dtype, false, stream);
}

extern "C" int uwc_w4_gated(const void* x, int64_t x_stride, int dtype, int M, const uint8_t* codes, const uint8_t* scales,
                            int F, int K, void* y, hipStream_t stream) {
  return call("uwc_w4_gated", W4Args{x, (long)x_stride, codes, scales, nullptr, y, M, F, F > 0x3fffffff ? F : 2 * F, K}, dtype, true, stream);
}
