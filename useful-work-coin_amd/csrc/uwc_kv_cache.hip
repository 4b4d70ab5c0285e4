// Appending to and reading from the paged 8-bit key/value cache (layout in uwc_kv.h).
//
//   append  per head row x of a new token at position p:
//             x' = x / sqrt(mean(x^2) + eps) * w            (q and k heads, where weights are given)
//             x'' = x' cos_p + (-hi, lo)(x') sin_p          (q and k heads)
//           q comes out in its own type. Keys and values go into their pages as
//             z = clamp(rint(x'' / s), -127, 127),  s = max(max |x''| over the page, 1e-8) / 127
//           with max over the page's new tokens; where it holds older ones s is at least their scale, and
//           they are rounded again, rint(z old / s), if it grew. An unchanged scale leaves them as they are
//           (rint(z s / s) = z), so a decode step writes its token alone.
//   read    value = z s of a range of tokens, rounded once to the output type; zeros in rows of no sequence.
//
// Bytes bound both where tokens are many (a prefill of 3890 tokens, 16 + 2 x 8 heads of 128: 60 MB in 15.8 us; 30000 tokens
// read back, 184 MB in 35.2 us, 5.2 TB/s), the chain cu -> table -> rows -> scale where they are few (one token 4.0 us,
// 96 of them 6.3). A head row of hd dims is held by hd / 16 lanes, each with 8 dims of the lower half and
// the 8 that rotate with them, so the rotation stays in a lane and loads are 16 bytes wide.
#include "uwc_kv.h"

namespace {

// |x| as bits: their order is that of the values, with NaN above everything, so a NaN reaches the scale.
__device__ __forceinline__ u32 abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

template <class T>
__device__ __forceinline__ void load16(const T* p, int half, float x[16]) {
  typedef typename kv_vec<T>::v8 v8;
  const v8 lo = *reinterpret_cast<const v8*>(p), hi = *reinterpret_cast<const v8*>(p + half);
#pragma unroll
  for (int i = 0; i < 8; i++) x[i] = (float)lo[i], x[8 + i] = (float)hi[i];
}

struct Turn {
  float c[16], s[16];
};

// cos and sin of position p for this lane's dims; a position outside the tables gives NaN.
__device__ __forceinline__ void load_turn(const float* cosb, const float* sinb, int positions, int p, int hd, int c, Turn& t) {
  const bool in = p >= 0 && p < positions;
  const long at = (long)(in ? p : 0) * hd + 8 * c;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    t.c[i] = cosb[at + i], t.c[8 + i] = cosb[at + hd / 2 + i];
    t.s[i] = sinb[at + i], t.s[8 + i] = sinb[at + hd / 2 + i];
  }
  if (!in)
#pragma unroll
    for (int i = 0; i < 16; i++) t.c[i] = kv_nan();
}

// x' and x'' above, for one head row held by LPH lanes.
template <int LPH>
__device__ __forceinline__ void norm_turn(float x[16], const float* w, int c, float eps, const Turn& t) {
  constexpr int HD = 16 * LPH;
  if (w) {
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; i++) ss += x[i] * x[i];
#pragma unroll
    for (int d = 1; d < LPH; d <<= 1) ss += __shfl_xor(ss, d, 64);
    const float r = __builtin_amdgcn_rsqf(ss * (1.0f / HD) + eps);
#pragma unroll
    for (int i = 0; i < 8; i++) {
      x[i] = x[i] * r * w[8 * c + i];
      x[8 + i] = x[8 + i] * r * w[HD / 2 + 8 * c + i];
    }
  }
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const float lo = x[i], hi = x[8 + i];
    x[i] = lo * t.c[i] - hi * t.s[i];
    x[8 + i] = hi * t.c[8 + i] + lo * t.s[8 + i];
  }
}

struct AppendArgs {
  const void* qkv;
  long stride;  // elements between rows of qkv
  KvRows rows;
  const int *ctx, *table;
  long table_stride;
  int width;
  const float *cosb, *sinb;
  int positions;
  const float *qn, *kn;
  float eps;
  int H, Hkv, lp;  // P = 1 << lp
  long pages;
  i8 *k, *v;
  float *ks, *vs;
  void* q;
  int units;  // bound on the pages touched
  bool deal;  // whole pages to one XCD
};

__device__ __forceinline__ long page_of(const AppendArgs& a, int b, int col) {
  const long id = col >= 0 && col < a.width ? a.table[b * a.table_stride + col] : -1;
  return id < a.pages ? id : -1;
}

// The q heads of one packed row, by one wave.
template <int HD, class T>
__device__ __forceinline__ void append_q(const AppendArgs& a, int row) {
  constexpr int LPH = HD / 16;
  const int lane = threadIdx.x & 63, c = lane % LPH;
  typedef typename kv_vec<T>::v8 v8;
  int b = row, i = 0;
  bool in = true;
  if (a.rows.cu) {  // sequences that end at or before this row come before its own
    int before = 0;
    for (int base = 0; base < a.rows.B; base += 64)
      before += __builtin_popcountll(__ballot(base + lane < a.rows.B && a.rows.cu[base + lane + 1] <= row));
    in = before < a.rows.B && row >= a.rows.cu[before < a.rows.B ? before : 0];
    b = in ? before : 0;
    i = row - a.rows.cu[b];
  }
  T* out = static_cast<T*>(a.q) + (long)row * a.H * HD;
  if (!in) {  // a row of no sequence
    for (int at = lane * 8; at < a.H * HD; at += 512) *reinterpret_cast<u4v*>(out + at) = u4v{0, 0, 0, 0};
    return;
  }
  const int ctx = a.ctx[b], pos = ctx + i;
  const bool bad = ctx < 0 || page_of(a, b, pos >> a.lp) < 0;
  Turn t;
  load_turn(a.cosb, a.sinb, a.positions, bad ? -1 : pos, HD, c, t);
  const T* x0 = static_cast<const T*>(a.qkv) + row * a.stride;
  for (int h = lane / LPH; h < a.H; h += 64 / LPH) {
    float x[16];
    load16(x0 + h * HD + 8 * c, HD / 2, x);
    norm_turn<LPH>(x, a.qn, c, a.eps, t);
    v8 lo, hi;
#pragma unroll
    for (int k = 0; k < 8; k++) lo[k] = (T)x[k], hi[k] = (T)x[8 + k];
    *reinterpret_cast<v8*>(out + h * HD + 8 * c) = lo;
    *reinterpret_cast<v8*>(out + h * HD + HD / 2 + 8 * c) = hi;
  }
}

__device__ __forceinline__ int quant8(float x, double rd) {
  return (int)fminf(fmaxf(rintf(uwc_div_rd(x, rd)), -127.0f), 127.0f);
}
// an older value under a grown scale: z old / s, the product and the quotient rounded once each
__device__ __forceinline__ int again8(int z, float old, double rd) { return (int)rintf(uwc_div_rd((float)z * old, rd)); }
__device__ __forceinline__ u32 again4(u32 w, float old, double rd) {
  u32 r = 0;
#pragma unroll
  for (int i = 0; i < 4; i++) r |= (u32)(again8((int)(i8)(w >> (8 * i)), old, rd) & 255) << (8 * i);
  return r;
}

// Pages that n tokens from position x on touch.
__device__ __forceinline__ int pages_of(int n, int x, int lp) {
  const int P = 1 << lp;
  return n == 0 || x < 0 ? 0 : (int)(((u32)(n + (x & (P - 1))) + P - 1) >> lp);
}

// The new tokens of one page of one kv head, keys (SIDE 0) or values (SIDE 1), by one workgroup.
// ROUNDS rounds of 256 / (hd / 16) tokens cover the page.
template <int HD, int ROUNDS, int SIDE, class T>
__device__ __forceinline__ void append_page(const AppendArgs& a, int unit, int h) {
  constexpr int LPH = HD / 16, PER = 256 / LPH;
  __shared__ u32 wmax[4];
  __shared__ __attribute__((aligned(16))) u8 img[SIDE ? HD * (PER * ROUNDS + 16) : 16];
  const int P = 1 << a.lp, tid = threadIdx.x, c = tid % LPH;
  KvUnit u{unit, 0, unit, 1, 0};
  if (!a.rows.cu) u.x = a.ctx[unit];
  else if (!kv_find(a.rows, a.ctx, unit, [&](int n, int x) KV_AI { return pages_of(n, x, a.lp); }, u)) return;
  const int b = u.b, j = u.j, ctx = u.x, n = u.n, lead = ctx & (P - 1);
  if (ctx < 0) return;
  const int first = j ? 0 : lead, i0 = j ? (j << a.lp) - lead : 0;
  const int row0 = u.row0 + i0;  // row of slot `first`
  int cnt = n - i0 < P - first ? n - i0 : P - first;
  const long id = page_of(a, b, (ctx >> a.lp) + j);
  if (id < 0) return;
  const long head = id * a.Hkv + h;
  float* sp = (SIDE ? a.vs : a.ks) + head;
  const float old = first ? *sp : 0.0f;

  float x[ROUNDS][16];
  u32 mx = 0;
#pragma unroll
  for (int r = 0; r < ROUNDS; r++) {
    const int s = r * PER + tid / LPH, row = row0 + s;
    if (s < cnt && row >= 0 && row < a.rows.T) {
      load16(static_cast<const T*>(a.qkv) + row * a.stride + (long)(a.H + SIDE * a.Hkv + h) * HD + 8 * c, HD / 2, x[r]);
      if constexpr (!SIDE) {
        Turn t;
        load_turn(a.cosb, a.sinb, a.positions, ctx + i0 + s, HD, c, t);
        norm_turn<LPH>(x[r], a.kn, c, a.eps, t);
      }
#pragma unroll
      for (int k = 0; k < 16; k++) {
        const u32 v = abs_bits(x[r][k]);
        mx = v > mx ? v : mx;
      }
    } else {
#pragma unroll
      for (int k = 0; k < 16; k++) x[r][k] = 0.0f;
    }
  }
  mx = kv_umax_wave(mx);
  if ((tid & 63) == 0) wmax[tid >> 6] = mx;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 4; w++) mx = wmax[w] > mx ? wmax[w] : mx;
  const u32 low = __float_as_uint(1e-8f);
  float s = __fdiv_rn(__uint_as_float(mx > low ? mx : low), 127.0f);
  if (abs_bits(old) > abs_bits(s)) s = old;
  if (tid == 0) *sp = s;
  const double rd = 1.0 / (double)s;
  const bool grew = first && !(s == old);

  if constexpr (!SIDE) {
    i8* kp = a.k + (head << a.lp) * HD;
    if (grew)
      for (int at = tid * 4; at < first * HD; at += 1024)
        *reinterpret_cast<u32*>(kp + at) = again4(*reinterpret_cast<const u32*>(kp + at), old, rd);
#pragma unroll
    for (int r = 0; r < ROUNDS; r++) {
      const int t = r * PER + tid / LPH;
      if (t >= cnt) continue;
      u32 w[4] = {0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < 16; k++) w[k >> 2] |= (u32)(quant8(x[r][k], rd) & 255) << (8 * (k & 3));
      i8* dst = kp + (first + t) * HD + 8 * c;
      *reinterpret_cast<uint2*>(dst) = uint2{w[0], w[1]};
      *reinterpret_cast<uint2*>(dst + HD / 2) = uint2{w[2], w[3]};
    }
  } else {
    i8* vp = a.v + (head << a.lp) * HD;
    if (cnt <= 8 && !grew) {  // a decode step: bytes straight to their places
#pragma unroll
      for (int r = 0; r < ROUNDS; r++) {
        const int t = r * PER + tid / LPH;
        if (t >= cnt) continue;
#pragma unroll
        for (int k = 0; k < 16; k++)
          vp[(long)((k >> 3) * (HD / 2) + 8 * c + (k & 7)) * P + first + t] = (i8)quant8(x[r][k], rd);
      }
      return;
    }
    // the page through LDS, its rows 16 bytes apart from a multiple of the banks: older tokens, new ones, zeros
    const int ld = P + 16;
    const int chunks = P >> 4, lc = a.lp - 4;
    for (int q = tid; q < HD * chunks; q += 256) {
      const int d = q >> lc, at = (q & (chunks - 1)) * 16;
      u4v w{0, 0, 0, 0};
      if (at < first) {
        w = *reinterpret_cast<const u4v*>(vp + (long)d * P + at);
        if (grew)
#pragma unroll
          for (int k = 0; k < 4; k++) w[k] = again4(w[k], old, rd);
      }
      *reinterpret_cast<u4v*>(img + d * ld + at) = w;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROUNDS; r++) {
      const int t = r * PER + tid / LPH;
      if (t >= P - first) continue;  // past the new tokens x is 0
#pragma unroll
      for (int k = 0; k < 16; k++)
        img[((k >> 3) * (HD / 2) + 8 * c + (k & 7)) * ld + first + t] = (u8)(quant8(x[r][k], rd) & 255);
    }
    __syncthreads();
    for (int q = tid; q < HD * chunks; q += 256) {
      const int d = q >> lc, at = (q & (chunks - 1)) * 16;
      *reinterpret_cast<u4v*>(vp + (long)d * P + at) = *reinterpret_cast<const u4v*>(img + d * ld + at);
    }
  }
}

// Workgroups: first `units` x 2 Hkv for the pages, then one for every four rows of q. Consecutive workgroups go to
// consecutive XCDs. Where sequences have several new tokens (deal), they are dealt such that all heads of a page, and 64
// consecutive rows of q, share an XCD and with it the rotation's rows in its L2 (a prefill of 3890 tokens in three
// sequences, 16 + 2 x 8 heads of 128: 17.3 us heads over the XCDs, 15.8 so; eights of pages and of rows in turn 18.1).
// With a token each a head stays on the XCD whose L2 the kernels that read it next look into (96 sequences, with the
// read-back 13.7 us, dealt 14.9).
template <int HD, int ROUNDS, class T>
__global__ __launch_bounds__(256) void kv_append_kernel(AppendArgs a) {
  const u32 sides = 2u * (u32)a.Hkv, pages = (u32)a.units * sides;
  if (blockIdx.x >= pages) {
    u32 i = blockIdx.x - pages;
    if (a.deal && i < (gridDim.x - pages) / 128 * 128) i = i / 128 * 128 + i % 8 * 16 + i % 128 / 8;
    const int row = __builtin_amdgcn_readfirstlane((int)(i * 4 + (threadIdx.x >> 6)));
    if (row < a.rows.T) append_q<HD, T>(a, row);
    return;
  }
  u32 unit = blockIdx.x / sides, sh = blockIdx.x % sides;
  if (a.deal && unit < ((u32)a.units & ~7u)) {
    const u32 r = blockIdx.x % (8 * sides);
    unit = blockIdx.x / (8 * sides) * 8 + r % 8, sh = r / 8;
  }
  if (sh < (u32)a.Hkv) append_page<HD, ROUNDS, 0, T>(a, (int)unit, (int)sh);
  else append_page<HD, ROUNDS, 1, T>(a, (int)unit, (int)sh - a.Hkv);
}

// past the caches: values that are written once (a prefix of 30000 tokens, 184 MB moved: 42.3 -> 36.0 us)
template <class V>
__device__ __forceinline__ void store16(void* p, V v) {
  __builtin_nontemporal_store(__builtin_bit_cast(u4v, v), reinterpret_cast<u4v*>(p));
}

struct ReadArgs {
  const i8 *k, *v;
  const float *ks, *vs;
  long pages;
  const int* table;
  long table_stride;
  int width;
  const int* start;
  KvRows rows;
  int Hkv, lp;
  void *ko, *vo;
};

// One page's tokens of one kv head; of a sequence that starts below 0 as many NaN. Workgroups past the last page take a
// page's worth of the rows of no sequence each, zeros. The first (HD / 8) (P / 16) pieces of work are its values', 16 tokens of 8 dims
// each: 16-byte loads along the tokens, 16-byte stores along the dims; the others its keys', 16 dims of a token.
template <int HD, class T>
__global__ __launch_bounds__(256) void kv_read_kernel(ReadArgs a) {
  typedef typename kv_vec<T>::v8 v8;
  const int P = 1 << a.lp, tid = threadIdx.x;
  const int h = blockIdx.x % a.Hkv;
  int unit = blockIdx.x / a.Hkv;
  KvUnit u;
  if (!kv_find(a.rows, a.start, unit, [&](int n, int x) KV_AI { return pages_of(n, x < 0 ? 0 : x, a.lp); }, u)) {
    const int from = a.rows.B && a.rows.cu[a.rows.B] > 0 ? a.rows.cu[a.rows.B] : 0;
    for (int q = tid; q < P * (HD / 8); q += 256) {
      const long r = from + ((long)unit << a.lp) + q / (HD / 8), at = (r * a.Hkv + h) * HD + q % (HD / 8) * 8;
      if (r >= a.rows.T) break;
      store16(static_cast<T*>(a.ko) + at, u4v{0, 0, 0, 0});
      store16(static_cast<T*>(a.vo) + at, u4v{0, 0, 0, 0});
    }
    return;
  }
  const int b = u.b, j = u.j, start = u.x < 0 ? 0 : u.x, n = u.n, lead = start & (P - 1);
  const int first = j ? 0 : lead, i0 = j ? (j << a.lp) - lead : 0, col = (start >> a.lp) + j;
  const int row0 = u.row0 + i0 - first;  // row of slot 0
  int lo = first, hi = first + (n - i0 < P - first ? n - i0 : P - first);
  lo = lo > -row0 ? lo : -row0;
  hi = hi < a.rows.T - row0 ? hi : a.rows.T - row0;
  long id = u.x >= 0 && col < a.width ? a.table[b * a.table_stride + col] : -1;
  const bool bad = id < 0 || id >= a.pages;
  if (bad) id = 0;
  const long head = id * a.Hkv + h;
  const float sk = bad ? kv_nan() : a.ks[head], sv = bad ? kv_nan() : a.vs[head];
  const i8 *kp = a.k + (head << a.lp) * HD, *vp = a.v + (head << a.lp) * HD;
  const int of_values = (HD / 8) * (P >> 4), all = of_values + P * (HD / 16);
  for (int q = tid; q < all; q += 256) {
    if (q < of_values) {
      const int d = q % (HD / 8) * 8, t0 = q / (HD / 8) * 16;
      if (t0 >= hi || t0 + 16 <= lo) continue;
      u4v w[8];
#pragma unroll
      for (int i = 0; i < 8; i++) w[i] = *reinterpret_cast<const u4v*>(vp + (long)(d + i) * P + t0);
      T* out = static_cast<T*>(a.vo) + ((long)(row0 + t0) * a.Hkv + h) * HD + d;
#pragma unroll
      for (int t = 0; t < 16; t++) {
        if (t0 + t < lo || t0 + t >= hi) continue;
        v8 y;
#pragma unroll
        for (int i = 0; i < 8; i++) y[i] = (T)((float)(i8)(w[i][t >> 2] >> (8 * (t & 3))) * sv);
        store16(out + (long)t * a.Hkv * HD, y);
      }
    } else {
      const int t = (q - of_values) / (HD / 16), c = (q - of_values) % (HD / 16) * 16;
      if (t < lo || t >= hi) continue;
      const u4v w = *reinterpret_cast<const u4v*>(kp + t * HD + c);
      v8 y[2];
#pragma unroll
      for (int i = 0; i < 16; i++) y[i >> 3][i & 7] = (T)((float)(i8)(w[i >> 2] >> (8 * (i & 3))) * sk);
      T* out = static_cast<T*>(a.ko) + ((long)(row0 + t) * a.Hkv + h) * HD + c;
      store16(out, y[0]);
      store16(out + 8, y[1]);
    }
  }
}

int check_cache(const char* fn, const void* k, const void* v, const void* ks, const void* vs, long pages, int page, int Hkv,
                int hd, int dtype) {
  if (!k || !v || !ks || !vs) return uwc_fail("%s: null cache", fn);
  if (pages <= 0 || pages > 0x7fffffff || Hkv <= 0 || Hkv > 65535) return uwc_fail("%s: bad pages=%ld Hkv=%d", fn, pages, Hkv);
  if (page != 16 && page != 32 && page != 64 && page != 128) return uwc_fail("%s: page %d not in {16, 32, 64, 128}", fn, page);
  if (hd != 32 && hd != 64 && hd != 128) return uwc_fail("%s: head_dim %d not in {32, 64, 128}", fn, hd);
  if (dtype != UWC_KV_BF16 && dtype != UWC_KV_FP16) return uwc_fail("%s: unknown dtype %d", fn, dtype);
  if (((uintptr_t)k | (uintptr_t)v) & 15) return uwc_fail("%s: k and v must be 16-byte aligned", fn);
  return UWC_OK;
}

// Pages that n packed rows of B sequences can touch: none more than its rows, at most two partial ones each.
long touched_bound(int B, int T, int page) {
  const long u = (long)T / page + 2L * B;
  return u < T ? u : T;
}

}  // namespace

extern "C" int uwc_kv_append(const void* qkv, int64_t qkv_stride, int dtype, int T, int B, const int32_t* cu,
                             const int32_t* ctx, const int32_t* table, int64_t table_stride, int width, const float* cosb,
                             const float* sinb, int positions, const float* q_norm, const float* k_norm, float eps, int H,
                             int Hkv, int hd, int page, int64_t pages, int8_t* k, int8_t* v, float* ks, float* vs, void* q,
                             hipStream_t stream) {
  const char* fn = "uwc_kv_append";
  if (int st = check_cache(fn, k, v, ks, vs, pages, page, Hkv, hd, dtype)) return st;
  if (T < 0 || B < 0 || H < 0 || width < 0 || table_stride < 0) return uwc_fail("%s: bad T=%d B=%d H=%d width=%d", fn, T, B, H, width);
  if (T == 0) return UWC_OK;
  if (!qkv || (B && (!ctx || !table)) || !cosb || !sinb || (!q && H) || positions <= 0) return uwc_fail("%s: null or empty arguments", fn);
  if (!cu && T != B) return uwc_fail("%s: without cu every sequence has one row (T=%d B=%d)", fn, T, B);
  if (qkv_stride % 8 || (((uintptr_t)qkv | (uintptr_t)q) & 15))
    return uwc_fail("%s: rows of qkv and q must be 16-byte aligned", fn);
  const long units = B == 0 ? 0 : cu ? touched_bound(B, T, page) : B;
  const long blocks = units * 2 * Hkv + ((H ? (long)T : 0) + 3) / 4;
  if (blocks > 0xFFFFFF) return uwc_fail("%s: too many tokens (%d) and heads (%d)", fn, T, Hkv);  // 2^32 threads
  const AppendArgs a{qkv, qkv_stride, {cu, B, T}, ctx, table, table_stride, width, cosb, sinb, positions, q_norm, k_norm, eps,
                     H, Hkv, __builtin_ctz((unsigned)page), pages, k, v, ks, vs, q, (int)units, T > 4L * B};
  const dim3 grid((unsigned)blocks), wg(256);
#define KV_APPEND(HD, ROUNDS)                                                                              \
  do {                                                                                                     \
    if (dtype == UWC_KV_BF16) hipLaunchKernelGGL((kv_append_kernel<HD, ROUNDS, __bf16>), grid, wg, 0, stream, a); \
    else hipLaunchKernelGGL((kv_append_kernel<HD, ROUNDS, _Float16>), grid, wg, 0, stream, a);             \
    return uwc_launch_status(fn);                                                                          \
  } while (0)
  if (hd == 32) KV_APPEND(32, 1);
  if (hd == 64) {
    if (page <= 64) KV_APPEND(64, 1);
    KV_APPEND(64, 2);
  }
  if (page <= 32) KV_APPEND(128, 1);
  if (page == 64) KV_APPEND(128, 2);
  KV_APPEND(128, 4);
}

extern "C" int uwc_kv_read(const int8_t* k, const int8_t* v, const float* ks, const float* vs, int64_t pages, int page, int Hkv,
                           int hd, const int32_t* table, int64_t table_stride, int width, const int32_t* start,
                           const int32_t* cu, int B, int rows, int dtype, void* ko, void* vo, hipStream_t stream) {
  const char* fn = "uwc_kv_read";
  if (int st = check_cache(fn, k, v, ks, vs, pages, page, Hkv, hd, dtype)) return st;
  if (rows < 0 || B < 0 || width < 0 || table_stride < 0) return uwc_fail("%s: bad rows=%d B=%d width=%d", fn, rows, B, width);
  if (rows == 0) return UWC_OK;
  if ((B && (!table || !start || !cu)) || !ko || !vo) return uwc_fail("%s: null arguments", fn);
  if (((uintptr_t)ko | (uintptr_t)vo) & 15) return uwc_fail("%s: outputs must be 16-byte aligned", fn);
  // one more than the sequences touch: what they leave of the bound may be a part of a page short of the other rows
  const long blocks = (touched_bound(B, rows, page) + 1) * Hkv;
  if (blocks > 0xFFFFFF) return uwc_fail("%s: too many tokens (%d) and heads (%d)", fn, rows, Hkv);
  const ReadArgs a{k, v, ks, vs, pages, table, table_stride, width, start, {cu, B, rows}, Hkv, __builtin_ctz((unsigned)page), ko, vo};
  const dim3 grid((unsigned)blocks), wg(256);
#define KV_READ(HD)                                                                                    \
  do {                                                                                                 \
    if (dtype == UWC_KV_BF16) hipLaunchKernelGGL((kv_read_kernel<HD, __bf16>), grid, wg, 0, stream, a); \
    else hipLaunchKernelGGL((kv_read_kernel<HD, _Float16>), grid, wg, 0, stream, a);                   \
    return uwc_launch_status(fn);                                                                      \
  } while (0)
  if (hd == 32) KV_READ(32);
  if (hd == 64) KV_READ(64);
  KV_READ(128);
}
