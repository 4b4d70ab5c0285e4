// Causal attention over the paged 8-bit key/value cache (layout in uwc_kv.h), grouped heads, optionally a
// sliding window with a few first tokens that stay visible:
//
//   s_ij = (q_i . kz_j) ks_j scale,  o_i = sum_j p_ij vz_j vs_j / sum_j p_ij,  p_ij = exp(s_ij - max)
//
// with kz, vz the cached bytes and ks, vs the scales of j's page. The scale of the values goes into the
// exponent: with t_ij = s_ij log2(e) + log2(vs_j) and m the row's maximum of t,
//
//   w_ij = 2^(t_ij - m) = p_ij vs_j (up to a factor of the row),  o_i = sum w_ij vz_j / sum w_ij (1 / vs_j)
//
// so the largest term of the numerator has weight 1 whatever the pages' scales are, and w can be rounded to
// fp16 (2^-11 relative; half as many bits again as bf16 would keep) for the matrix cores. The denominator is summed
// in fp32 from the unrounded w. kz and vz are exact in fp16. So is q: each row is scaled by a power of two
// to a maximum in [2^13, 2^14), which only drops bits 2^-38 below the row's maximum.
//
// The rows of a kv head are its (token, head of the group) pairs, so the heads of a group share each key.
// Scores are made transposed, S^T = K Q^T: a lane then holds keys of one row, and those registers are, lane
// by lane, the operand of O^T = V^T P^T; P never leaves them. The keys of a tile are dealt to the rows of K's
// operand so that a lane gets 16 consecutive tokens: one granule, one scale, one 16-byte piece of V's rows.
//
// m is not the row's maximum itself but at least 7 below it, and it only moves when some row's new maximum exceeds it by
// more than 15: the largest w lies in [2^7, 2^15], near the top of fp16, and most tiles neither exchange maxima between
// lanes nor rescale O. Weights down to 2^-21 of the row's largest then keep fp16's 11 bits, smaller ones are off by at most 2^-32
// of it: the long flat tail behind one key that is far ahead (a first token that all rows look at, often with values
// near 0) still counts. With the largest w at 1, 9000 keys 18 nats behind one of value 0 came out as 0.
#include <type_traits>

#include "uwc_kv.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

struct AttendArgs {
  const i8 *k, *v;
  const float *ks, *vs;
  long pages;
  const void* q;
  long q_stride;  // elements between tokens
  const int* table;
  long table_stride;
  int width;
  const int* lens;
  KvRows rows;
  int H, Hkv, G, lp;
  int window, sinks;
  float c;  // scale * log2(e)
  int units, splits, tps, fold;
  void* o;
  float* po;   // splits x T H x hd: unnormalised outputs, when splits > 1
  float2* ml;  // splits x T H: their m and denominator
};

constexpr float KV_LOWEST = -3e38f;  // m of a row that has seen nothing: differences from it stay numbers
constexpr float KV_BELOW = 7.0f, KV_MOVE = 15.0f;

// bytes of w as four fp16: 0x6400 | (x + 128) is 1024 + x + 128 in fp16, and subtracting 1152 is exact
__device__ __forceinline__ void to_half4(u32 w, h2v& a, h2v& b) {
  const u32 u = w ^ 0x80808080u;
  const h2v k = {(_Float16)-1152.0f, (_Float16)-1152.0f};
  a = __builtin_bit_cast(h2v, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) + k;
  b = __builtin_bit_cast(h2v, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) + k;
}
__device__ __forceinline__ h8v to_half8(u32 w0, u32 w1) {
  h2v a, b, c, d;
  to_half4(w0, a, b);
  to_half4(w1, c, d);
  return h8v{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

__device__ __forceinline__ float max_xor16(float v) { return fmaxf(v, __shfl_xor(v, 16, 64)); }
__device__ __forceinline__ float max_xor32(float v) { return fmaxf(v, __shfl_xor(v, 32, 64)); }

// The keys that the rows of one tile of queries can see, in tiles of 64: those of the first tokens that stay
// visible, then lt .. last.
struct Span {
  int p_lo, p_hi;  // positions of the first and the last query
  int lo;          // first key of the window of p_lo
  int st, lt, n;
  __device__ __forceinline__ int tile(int t) const { return t < st ? t : lt + t - st; }
};
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ Span span_of(const AttendArgs& a, int p_lo, int p_hi) {
  Span s;
  s.p_lo = p_lo = uniform(p_lo), s.p_hi = p_hi = uniform(p_hi);
  s.lo = a.window && p_lo >= a.window ? p_lo - a.window + 1 : 0;
  s.lt = s.lo >> 6;
  // Lengths and sinks far past the table's last page (there are no keys: NaN) take no more tiles than it needs to show.
  const long end = ((long)a.width << a.lp) >> 6, last = (end > s.lt ? end : s.lt) + ((p_hi - p_lo) >> 6) + 1;
  const int first = (a.sinks + 63) >> 6, head = first < s.lt ? first : s.lt;
  s.st = head <= end ? head : (int)end + 1;
  s.n = p_hi < 0 ? 0 : s.st + (int)((p_hi >> 6) < last ? p_hi >> 6 : last) - s.lt + 1;
  return s;
}
// Does any row see a key of key0 .. key0 + count - 1? Do all rows see all of them?
__device__ __forceinline__ bool any_seen(const AttendArgs& a, const Span& s, int key0, int count) {
  return key0 <= s.p_hi && (key0 + count > s.lo || key0 < a.sinks);
}
__device__ __forceinline__ bool all_seen(const AttendArgs& a, const Span& s, int key0, int count) {
  return key0 + count - 1 <= s.p_lo && (!a.window || key0 > s.p_hi - a.window || key0 + count <= a.sinks);
}
// Bit j: does a query at pos see key key0 + j?
__device__ __forceinline__ u32 seen32(const AttendArgs& a, int pos, int key0) {
  auto below = [](int n) KV_AI { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1; };
  const u32 m = below(pos - key0 + 1);
  return a.window ? m & (~below(pos - a.window + 1 - key0) | below(a.sinks - key0)) : m;
}
// v where bit j of m is set, else -inf
__device__ __forceinline__ float pick(u32 m, int j, float v) {
  const u32 t = (u32)__builtin_amdgcn_sbfe((int)m, j, 1);
  return __uint_as_float((t & __float_as_uint(v)) | (~t & 0xff800000u));
}

// The page of the granule that starts at key0: 0 where no row needs it, -1 where one does and there is none.
__device__ __forceinline__ int page_of(const AttendArgs& a, const Span& s, int b, int key0) {
  if (!any_seen(a, s, key0, 16)) return 0;
  const int col = key0 >> a.lp;
  const int id = col < a.width ? a.table[b * a.table_stride + col] : -1;
  return id < a.pages ? id : -1;
}

// Where a unit's rows lie: `r0` its first row in its sequence, n G rows of the sequence in all.
struct Unit {
  int b, r0, rows, row0, len;
  __device__ __forceinline__ int pos(const AttendArgs& a, int r) const { return len - rows / a.G + r / a.G; }
};

// Unit number u of tiles of M rows; false past the last (u then counts on from there).
__device__ __forceinline__ bool unit_of(const AttendArgs& a, int& u, int M, Unit& x) {
  if (a.rows.cu) {
    KvUnit k;
    if (!kv_find(a.rows, a.lens, u, [&](int n, int) KV_AI { return (int)(((long)n * a.G + M - 1) / M); }, k)) return false;
    x.b = k.b, x.r0 = k.j * M, x.rows = k.n * a.G, x.row0 = k.row0, x.len = k.x;
  } else {
    const int per = (a.G + M - 1) / M;
    x.b = uniform(u / per), x.r0 = uniform(u % per * M), x.rows = a.G, x.row0 = x.b, x.len = uniform(a.lens[x.b]);
  }
  return true;
}

// Row r of a unit: its packed row t (-1 outside) and head; row = t H + head.
struct Place {
  int t, head;
  __device__ __forceinline__ long row(const AttendArgs& a) const { return t < 0 ? -1 : (long)t * a.H + head; }
};
__device__ __forceinline__ Place place_of(const AttendArgs& a, const Unit& x, int r, int h) {
  const int i = r / a.G, t = x.row0 + i;
  return Place{r < x.rows && t >= 0 && t < a.rows.T ? t : -1, h * a.G + r - i * a.G};
}

template <class T, int N>
__device__ __forceinline__ void store_row(T* dst, const float* v) {
  typedef T tv __attribute__((ext_vector_type(N)));
  tv y;
#pragma unroll
  for (int i = 0; i < N; i++) y[i] = (T)v[i];
  *reinterpret_cast<tv*>(dst) = y;
}

// One output row's dims d .. d + N - 1: final, or this split's part.
template <int HD, int N, class T>
__device__ __forceinline__ void put(const AttendArgs& a, long row, int split, int d, const float* o, float m, float l) {
  if (a.splits == 1) {
    float y[N];
    const float r = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int i = 0; i < N; i++) y[i] = o[i] * r;
    store_row<T, N>(static_cast<T*>(a.o) + row * HD + d, y);
  } else {
    const long at = (long)split * a.rows.T * a.H + row;
#pragma unroll
    for (int i = 0; i < N; i += 2) *reinterpret_cast<float2*>(a.po + at * HD + d + i) = float2{o[i], o[i + 1]};
    if (d == 0) a.ml[at] = float2{m, l};
  }
}

// Rows of no sequence come out as zeros: unit u past the last one takes its share of those from cu[B] on.
template <int HD, class T>
__device__ __forceinline__ void zero_rows(const AttendArgs& a, int u, int M, int h, int split) {
  const int from = a.rows.cu[a.rows.B] < 0 ? 0 : a.rows.cu[a.rows.B];
  float z[HD / 16] = {};
  for (int i = threadIdx.x; i < M * 16; i += blockDim.x) {
    const long r = (long)u * M + i / 16, t = from + r / a.G;
    if (t < a.rows.T) put<HD, HD / 16, T>(a, t * a.H + h * a.G + r % a.G, split, (i & 15) * (HD / 16), z, KV_LOWEST, 0.0f);
  }
}

// ------------------------------------------------------------------ few rows
// A workgroup takes 16 RB rows of one kv head and a run of 64-key tiles, its four waves every fourth tile
// each, straight from memory into registers; their results meet in LDS. Bytes bound it: a tile of heads of 128 is 16 KiB
// against 350 VALU and 32 matrix instructions of a wave, a quarter of what its SIMD could do meanwhile, and two
// workgroups to a CU keep 128 KiB on their way (the next tile's keys are loaded when this one's are used up, its values
// after the products). 48 sequences of 1500 to 12000 tokens, 8 kv heads of 128: 723 MB in 146 us, 4.96 TB/s; one of
// 131072: 268 MB in 54, 4.94, the join included; a copy of 4 GiB moves 4.8 here, a streaming sum of rows reads 6.45. Loads
// past the caches: 151 and 59.
template <int HD>
struct Tile {
  static constexpr int KC = HD >= 64 ? HD / 64 : 1;  // 16-byte pieces (8-byte at HD = 32) of a key row in a lane
  u4v k[4][KC];
  u4v v[HD / 16];
  float ks, vs;
};

template <int HD>
__device__ __forceinline__ void load_keys(const AttendArgs& a, int kt, int h, int id, Tile<HD>& t) {
  const int lane = threadIdx.x & 63, g = lane >> 4, m = lane & 15, mask = (1 << a.lp) - 1;
  const int idm = __shfl(id, (m >> 2) * 16, 64);  // the page of the granule this lane's key rows lie in
  const i8* kp = a.k + ((((long)(idm < 0 ? 0 : idm) * a.Hkv + h) << a.lp) + ((kt * 64 + 16 * (m >> 2)) & mask)) * HD;
#pragma unroll
  for (int bl = 0; bl < 4; bl++) {
    const i8* row = kp + (4 * bl + (m & 3)) * HD;
    if constexpr (HD == 32) {
      const uint2 w = *reinterpret_cast<const uint2*>(row + 8 * g);
      t.k[bl][0] = u4v{w.x, w.y, 0, 0};
    } else {
#pragma unroll
      for (int c = 0; c < HD / 64; c++) t.k[bl][c] = *reinterpret_cast<const u4v*>(row + 64 * c + 16 * g);
    }
  }
  const bool used = id >= 0;
  const long at = (long)(used ? id : 0) * a.Hkv + h;
  t.ks = used ? a.ks[at] : kv_nan();
  t.vs = a.vs[at];
}

template <int HD>
__device__ __forceinline__ void load_values(const AttendArgs& a, int kt, int h, int id, Tile<HD>& t) {
  const int lane = threadIdx.x & 63, g = lane >> 4, m = lane & 15, P = 1 << a.lp;
  const i8* vp = a.v + (((long)(id < 0 ? 0 : id) * a.Hkv + h) << a.lp) * HD + ((kt * 64 + 16 * g) & (P - 1));
#pragma unroll
  for (int db = 0; db < HD / 16; db++) t.v[db] = *reinterpret_cast<const u4v*>(vp + (long)(16 * db + m) * P);
}

// 8 consecutive dims of a query row as fp16 scaled by 2^e
template <class T>
__device__ __forceinline__ h8v scaled_q(const typename kv_vec<T>::v8& x, int e) {
  h8v y;
#pragma unroll
  for (int i = 0; i < 8; i++) y[i] = (_Float16)__builtin_amdgcn_ldexpf((float)x[i], e);
  return y;
}
// the exponent that takes a row's maximum (as bits of |x|) into [2^13, 2^14); 0 for rows of zeros, infinities, NaN
__device__ __forceinline__ int q_shift(u32 top) {
  const int e = (int)(top >> 23);
  return top == 0 || e == 255 ? 0 : 13 - (e - 127);
}

template <int HD, int RB, class T>
__global__ __launch_bounds__(256) void kv_attend_few_kernel(AttendArgs a) {
  typedef typename kv_vec<T>::v8 v8;
  constexpr int M = 16 * RB, KS = HD / 32, DB = HD / 16, LDO = HD + 4;
  __shared__ float sm[4][M], sl[4][M];
  __shared__ float so[4][16][LDO];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, m16 = lane & 15;
  const int h = blockIdx.x % a.Hkv, rest = blockIdx.x / a.Hkv, split = rest % a.splits;
  int u = rest / a.splits;
  Unit x;
  if (!unit_of(a, u, M, x)) {
    zero_rows<HD, T>(a, u, M, h, split);
    return;
  }

  // queries: lane (row m16, g) holds, of every 32-dim step, the 8 dims that its pieces of a key row hold
  h8v q[RB][KS];
  float A[RB];
  int pos[RB];
#pragma unroll
  for (int rb = 0; rb < RB; rb++) {
    const int r = x.r0 + rb * 16 + m16;
    const Place at = place_of(a, x, r, h);
    pos[rb] = at.t < 0 ? -1 : x.pos(a, r);
    const T* qp = static_cast<const T*>(a.q) + (at.t < 0 ? 0 : at.t * a.q_stride + at.head * HD);
    v8 w[KS];
    u32 top = 0;
#pragma unroll
    for (int s = 0; s < KS; s++) {
      const int d = HD == 32 ? 8 * g : 64 * (s >> 1) + 16 * g + 8 * (s & 1);
      w[s] = *reinterpret_cast<const v8*>(qp + d);
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const u32 bits = __float_as_uint((float)w[s][i]) & 0x7fffffffu;
        top = bits > top ? bits : top;
      }
    }
#pragma unroll
    for (int d = 16; d < 64; d <<= 1) {
      const u32 o = (u32)__shfl_xor((int)top, d, 64);
      top = o > top ? o : top;
    }
    const int e = q_shift(top);
    A[rb] = __builtin_amdgcn_ldexpf(a.c, -e);
#pragma unroll
    for (int s = 0; s < KS; s++) q[rb][s] = scaled_q<T>(w[s], e);
  }

  f32x4 o[RB][DB];
  float mr[RB], l[RB];
#pragma unroll
  for (int rb = 0; rb < RB; rb++) {
    mr[rb] = KV_LOWEST, l[rb] = 0.0f;
#pragma unroll
    for (int db = 0; db < DB; db++) o[rb][db] = f32x4{0, 0, 0, 0};
  }

  const int last_r = x.r0 + M < x.rows ? x.r0 + M - 1 : x.rows - 1;
  const Span sp = span_of(a, x.pos(a, x.r0), x.pos(a, last_r));
  const int t0 = split * a.tps + wave, t1 = split + 1 == a.splits ? sp.n : min(sp.n, (split + 1) * a.tps);
  Tile<HD> t;
  int id = 0, nid = 0;
  if (t0 < t1) {
    id = page_of(a, sp, x.b, sp.tile(t0) * 64 + 16 * g);
    load_keys<HD>(a, sp.tile(t0), h, id, t);
    load_values<HD>(a, sp.tile(t0), h, id, t);
    if (t0 + 4 < t1) nid = page_of(a, sp, x.b, sp.tile(t0 + 4) * 64 + 16 * g);
  }
  for (int it = t0; it < t1; it += 4) {
    const int kt = sp.tile(it), next = sp.tile(it + 4);
    const bool more = it + 4 < t1;
    f32x4 s[RB][4];
#pragma unroll
    for (int bl = 0; bl < 4; bl++) {
#pragma unroll
      for (int rb = 0; rb < RB; rb++) s[rb][bl] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int ks = 0; ks < KS; ks++) {
        const u4v w = t.k[bl][ks >> 1];
        const h8v kf = ks & 1 ? to_half8(w[2], w[3]) : to_half8(w[0], w[1]);
#pragma unroll
        for (int rb = 0; rb < RB; rb++) s[rb][bl] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, q[rb][ks], s[rb][bl], 0, 0, 0);
      }
    }
    const float ks = t.ks, vs = fmaxf(t.vs, 0x1p-90f);
    const float lv = t.vs != t.vs ? kv_nan() : __builtin_amdgcn_logf(vs), rv = __builtin_amdgcn_rcpf(vs);
    if (more) load_keys<HD>(a, next, h, nid, t);
    const bool whole = all_seen(a, sp, kt * 64, 64);
    h8v p[RB][2];
#pragma unroll
    for (int rb = 0; rb < RB; rb++) {
      const float Ak = A[rb] * ks;
      float e[16], top = -__builtin_inff();
#pragma unroll
      for (int i = 0; i < 16; i++) e[i] = __builtin_fmaf(s[rb][i >> 2][i & 3], Ak, lv);
      if (!whole) {
        const u32 m = seen32(a, pos[rb], kt * 64 + 16 * g);
#pragma unroll
        for (int i = 0; i < 16; i++) e[i] = pick(m, i, e[i]);
      }
#pragma unroll
      for (int i = 0; i < 16; i++) top = fmaxf(top, e[i]);
      if (__any(top > mr[rb] + KV_MOVE)) {
        const float to = fmaxf(mr[rb], max_xor32(max_xor16(top)) - KV_BELOW);
        const float f = __builtin_amdgcn_exp2f(mr[rb] - to);
        mr[rb] = to;
        l[rb] *= f;
#pragma unroll
        for (int db = 0; db < DB; db++) o[rb][db] *= f;
      }
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 16; i++) {
        e[i] = __builtin_amdgcn_exp2f(e[i] - mr[rb]);
        sum += e[i];
        p[rb][i >> 3][i & 7] = (_Float16)e[i];
      }
      l[rb] = sum == 0.0f ? l[rb] : __builtin_fmaf(sum, rv, l[rb]);  // a granule nobody sees may have any scale
    }
#pragma unroll
    for (int db = 0; db < DB; db++) {
      const u4v w = t.v[db];
      const h8v v0 = to_half8(w[0], w[1]), v1 = to_half8(w[2], w[3]);
#pragma unroll
      for (int rb = 0; rb < RB; rb++) {
        o[rb][db] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, p[rb][0], o[rb][db], 0, 0, 0);
        o[rb][db] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, p[rb][1], o[rb][db], 0, 0, 0);
      }
    }
    if (more) {
      load_values<HD>(a, next, h, nid, t);
      id = nid;
      if (it + 8 < t1) nid = page_of(a, sp, x.b, sp.tile(it + 8) * 64 + 16 * g);
    }
  }

#pragma unroll
  for (int rb = 0; rb < RB; rb++) {
    l[rb] += __shfl_xor(l[rb], 16, 64);
    l[rb] += __shfl_xor(l[rb], 32, 64);
    if (g == 0) sm[wave][rb * 16 + m16] = mr[rb], sl[wave][rb * 16 + m16] = l[rb];
  }
  __syncthreads();
#pragma unroll
  for (int rb = 0; rb < RB; rb++) {
    const int r = rb * 16 + m16;
    const float top = fmaxf(fmaxf(sm[0][r], sm[1][r]), fmaxf(sm[2][r], sm[3][r]));
    const float f = __builtin_amdgcn_exp2f(mr[rb] - top);
    if (rb) __syncthreads();
#pragma unroll
    for (int db = 0; db < DB; db++) *reinterpret_cast<f32x4*>(&so[wave][m16][16 * db + 4 * g]) = o[rb][db] * f;
    __syncthreads();
    constexpr int N = HD / 16;
    const int ro = tid >> 4, d = (tid & 15) * N, rr = rb * 16 + ro;
    const long row = place_of(a, x, x.r0 + rr, h).row(a);
    if (row >= 0) {
      float y[N], tm = fmaxf(fmaxf(sm[0][rr], sm[1][rr]), fmaxf(sm[2][rr], sm[3][rr])), tl = 0.0f;
#pragma unroll
      for (int w = 0; w < 4; w++) tl += sl[w][rr] * __builtin_amdgcn_exp2f(sm[w][rr] - tm);
#pragma unroll
      for (int i = 0; i < N; i++) y[i] = so[0][ro][d + i] + so[1][ro][d + i] + so[2][ro][d + i] + so[3][ro][d + i];
      put<HD, N, T>(a, row, split, d, y, tm, tl);
    }
  }
}

// ------------------------------------------------------------------ many rows
// A workgroup of NW waves takes 32 NW rows of one kv head; the keys and values of a 64-key tile are turned into
// fp16 once per workgroup, in LDS, and every wave multiplies its own 32 rows with them on 32 x 32 x 16 matrix
// instructions. A step has two halves with a barrier after each: the weights of a tile (VALU: 32 exponentials of 16
// cycles each and some 130 other instructions per wave, about 1200 cycles), and its product with V and the next tile's
// scores (32 matrix instructions, 1024 cycles, fed by LDS reads six ahead), between which the next bytes are
// converted, written to LDS and loaded. With eight waves the two of a SIMD take turns at the halves, a barrier apart.
//
// Four waves (two workgroups to a CU) keep two stages of keys and of values: in the second half of step i, which reads
// keys i + 1 and values i, the keys of tile i + 2 take the place of keys i and the values of tile i + 1 that of values
// i - 1, both last read before the barriers between. Eight waves keep four stages of either, as the waves that are half a
// step behind still read values i when the others are a half past them, and write tile i + 2 in step i's second half.
//
// LDS rows hold 16-byte pieces (8 fp16), piece c of row r at c ^ swz(r), such that 16 lanes, which LDS serves at once,
// hit all of its 64 banks: 16 rows of an operand that are read, two key rows or four value rows that are written. K's operand row m is key 16 (m >> 4) + 8 (m >> 2 & 1) + 4 (m >> 3 & 1) +
// (m & 3) of its 32: the scores of lane half hf are then keys 16 n + 8 hf + i, the 8 k slots of V's product n.
//
// Measured: 4096 tokens over 32768, 16 heads of 128, 964 to 1031 us by box = 1070 to 1000 TFLOP/s, at a clock that the
// load drives down to about 1.88 GHz (an fp16 product of 16384^3 reaches 1263 to 1328 here): matrix units busy 52% of its
// cycles, VALU 59%. 6000 tokens under a window of 1024, heads of 64: 47 us (three workgroups to a CU, 168 registers; two
// 58 us); neither unit is full, VALU 50% and matrix units 20% of the cycles, with 1.75 waves to a SIMD on average of the
// three that fit: waves that wait at the barriers, and workgroups that have ended while others go on.
__device__ __forceinline__ int key_row(int key) { return (key & ~12) | ((key & 4) << 1) | ((key & 8) >> 1); }
template <int HD>
__device__ __forceinline__ int k_piece(int r, int c) {  // of rows of HD fp16
  if (HD == 32) return r * 4 + (c ^ ((r >> 1) & 3));
  return HD == 128 ? r * 16 + (c ^ (r & 15)) : r * 8 + (c ^ ((r ^ (r >> 3 & 3)) & 7));
}
__device__ __forceinline__ int v_piece(int r, int c) { return r * 8 + (c ^ ((r ^ (r >> 3 & 3)) & 7)); }

// The weights of one 32-row block for a tile of 64 keys: p the operands of V's products, m the running maximum and
// l this lane's part of the denominator brought up to date, o rescaled where m moved.
template <int DB>
__device__ __forceinline__ void softmax_tile(const AttendArgs& a, f16v s[2], float A, int pos, bool whole, int key0,
                                             const float4* meta, f16v* o, float& mr, float& l, h8v p[4]) {
  // 2^(s Ak + lk - m) is the weight; Ak > 0, so the maximum of s gives that of the exponent
  float Ak[4], lk[4], rv[4], top = -__builtin_inff();
#pragma unroll
  for (int n = 0; n < 4; n++) {
    const float4 mt = meta[n];
    Ak[n] = A * mt.x, lk[n] = mt.y, rv[n] = mt.z;
  }
  if (!whole) {
    const u32 seen[2] = {seen32(a, pos, key0), seen32(a, pos, key0 + 32)};
#pragma unroll
    for (int n = 0; n < 4; n++) {
#pragma unroll
      for (int i = 0; i < 8; i++) s[n >> 1][8 * (n & 1) + i] = pick(seen[n >> 1], 16 * (n & 1) + i, s[n >> 1][8 * (n & 1) + i]);
      const bool some = seen[n >> 1] & 0xffu << 16 * (n & 1);
      // -inf has to stay -inf, also under a scale of 0, and under any scale of keys this row does not see
      Ak[n] = !some ? 1.0f : Ak[n] == 0.0f ? 0x1p-126f : Ak[n];
      lk[n] = some ? lk[n] : 0.0f;
    }
  }
#pragma unroll
  for (int n = 0; n < 4; n++) {
    float g = s[n >> 1][8 * (n & 1)];
#pragma unroll
    for (int i = 1; i < 8; i++) g = fmaxf(g, s[n >> 1][8 * (n & 1) + i]);
    top = fmaxf(top, __builtin_fmaf(g, Ak[n], lk[n]));
  }
  if (__any(top > mr + KV_MOVE)) {
    const float to = fmaxf(mr, max_xor32(top) - KV_BELOW);
    const float f = __builtin_amdgcn_exp2f(mr - to);
    mr = to;
    l *= f;
#pragma unroll
    for (int db = 0; db < DB; db++) o[db] *= f;
  }
#pragma unroll
  for (int n = 0; n < 4; n++) {
    const float b = lk[n] - mr;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n >> 1][8 * (n & 1) + i], Ak[n], b));
      sum += w;
      p[n][i] = (_Float16)w;
    }
    l = sum == 0.0f ? l : __builtin_fmaf(sum, rv[n], l);  // keys nobody sees may have any scale
  }
}

typedef h8v __attribute__((address_space(3)))* lds_h8;
__device__ __forceinline__ u32 lds_addr(const h8v* q) { return (u32)(uintptr_t)(void __attribute__((address_space(3)))*)q; }
__device__ __forceinline__ void lds_put(u32 a, h8v v) { *(lds_h8)(uintptr_t)a = v; }

// LDS operations done, then everyone's; loads from memory stay on their way
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

template <int HD, int NW, class T>
__global__ __launch_bounds__(64 * NW, HD <= 64 ? 3 : 2) void kv_attend_many_kernel(AttendArgs a) {
  typedef typename kv_vec<T>::v8 v8;
  constexpr bool TURNS = NW == 8;
  constexpr int M = 32 * NW, NT = 64 * NW, KS = HD / 16, DB = HD / 32, STAGES = TURNS ? 4 : 2;
  constexpr int ROOM = 64 * HD / 8;  // pieces of fp16 of a tile's keys, and of its values
  __shared__ __attribute__((aligned(256))) h8v sk[STAGES * ROOM], sv[STAGES * ROOM];
  __shared__ float4 meta[32][4];  // ks, log2(vs), 1 / vs of a tile's granules
  __shared__ int ids[32][4];      // their pages
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), hf = lane >> 5, m32 = lane & 31;
  const int h = blockIdx.x % a.Hkv, rest = blockIdx.x / a.Hkv, split = rest % a.splits;
  // The last rows of a sequence see the most keys: first. Where all workgroups fit at once (fold), the second half goes
  // from the fewest keys up, so that a CU's two make up for each other.
  const int nth = rest / a.splits, half = a.units >> 1;
  int u = a.fold && nth >= half ? nth - half : a.units - 1 - nth;
  Unit x;
  if (!unit_of(a, u, M, x)) {
    zero_rows<HD, T>(a, u, M, h, split);
    return;
  }

  const int r = x.r0 + wave * 32 + m32;
  const Place mine = place_of(a, x, r, h);
  const int pos = mine.t < 0 ? -1 : x.pos(a, r);
  const T* qp = static_cast<const T*>(a.q) + (mine.t < 0 ? 0 : mine.t * a.q_stride + mine.head * HD);

  const int last_r = x.r0 + M < x.rows ? x.r0 + M - 1 : x.rows - 1;
  const Span sp = span_of(a, x.pos(a, x.r0), x.pos(a, last_r));
  Span of_wave = sp;  // what the wave's own rows see
  of_wave.p_lo = uniform(x.pos(a, min(x.r0 + wave * 32, last_r)));
  of_wave.p_hi = uniform(x.pos(a, min(x.r0 + wave * 32 + 31, last_r)));
  const int t0 = split * a.tps, n = uniform((split + 1 == a.splits ? sp.n : min(sp.n, (split + 1) * a.tps)) - t0);

  // The pages and scales of 16 tiles at a time, by the first wave, a lane a granule: the table is read at a step
  // that starts 16 tiles, the scales some steps later, and when 8 are left both are put into LDS for the next 16.
  const int* const pages_of = a.table + x.b * a.table_stride;
  struct Granule {
    int page;  // -1: needed and not there; -2: nobody looks
    float ks, vs;
  };
  auto load_page = [&](int t, Granule& c) KV_AI {
    t += lane >> 2;
    const int key0 = sp.tile(t0 + t) * 64 + 16 * (lane & 3), col = key0 >> a.lp;
    c.page = -2;
    if (t < n && any_seen(a, sp, key0, 16)) c.page = col < a.width ? max(pages_of[col], -1) : -1;
  };
  auto load_scales = [&](Granule& c) KV_AI {
    c.page = c.page < a.pages ? c.page : -1;
    const long at = (long)max(c.page, 0) * a.Hkv + h;
    c.ks = a.ks[at], c.vs = a.vs[at];
  };
  auto put_granule = [&](int t, const Granule& c) KV_AI {
    const float vs = fmaxf(c.vs, 0x1p-90f);
    const float4 m{c.page < 0 ? kv_nan() : c.ks, c.vs != c.vs ? c.vs : __builtin_amdgcn_logf(vs), __builtin_amdgcn_rcpf(vs), 0};
    meta[(t + (lane >> 2)) & 31][lane & 3] = c.page == -2 ? float4{0, 0, 0, 0} : m;
    ids[(t + (lane >> 2)) & 31][lane & 3] = c.page;
  };

  Granule next{-2, 0, 0};
  if (wave == 0) {
    load_page(0, next);
    next.page = next.page < a.pages ? next.page : -1;
    ids[lane >> 2][lane & 3] = next.page;
  }

  // The 16-byte pieces of a tile's keys, then those of its values, dealt to the threads; a wave's k-th
  // pieces are all of one kind.
  constexpr int PIECES = 64 * HD / 16, PER = 2 * PIECES > NT ? 2 * PIECES / NT : 1;
  const int mask = (1 << a.lp) - 1;
  const bool busy = 2 * PIECES >= NT || tid < 2 * PIECES;
  const u32 page_bytes = ((u32)a.Hkv << a.lp) * HD;
  const i8 *kh = a.k + ((long)h << a.lp) * HD, *vh = a.v + ((long)h << a.lp) * HD;
  u32 poff[PER], dst[PER];  // where a piece lies in a page, the tile's first key apart, and its first half in LDS
  int gran[PER];            // its granule
  auto of_values = [&](int k) KV_AI { return PER > 1 ? k >= PER / 2 : uniform(tid >= PIECES); };
#pragma unroll
  for (int k = 0; k < PER; k++) {
    const int p = (tid + k * NT) % PIECES, key = p / (HD / 16), c = p % (HD / 16), d = p >> 2, tg = p & 3;
    const bool values = of_values(k);
    poff[k] = values ? (u32)((d << a.lp) + ((16 * tg) & mask)) : (u32)((key & mask) * HD + 16 * c);
    gran[k] = values ? tg : key >> 4;
    dst[k] = lds_addr(values ? sv + v_piece(d, 2 * tg) : sk + k_piece<HD>(key_row(key), 2 * c));
  }

  h8v q[KS];
  float A = 0.0f;
  f16v o[DB];
  float mr = KV_LOWEST, l = 0.0f;
#pragma unroll
  for (int db = 0; db < DB; db++)
#pragma unroll
    for (int i = 0; i < 16; i++) o[db][i] = 0.0f;
  if (n > 0) {
    u4v st[PER];
    int idp[PER];  // the pages of the next pieces to be loaded
    h8v p[4];
    f16v s[2];
    auto load_id = [&](int i, int k) KV_AI { idp[k] = ids[i & 31][gran[k]]; };
    auto load_piece = [&](int i, int k) KV_AI {
      const int off = (sp.tile(t0 + i) * 64) & mask;  // pages of 64 and fewer start with a tile
      st[k] = *reinterpret_cast<const u4v*>((of_values(k) ? vh + off : kh + off * HD) + ((u64)(u32)max(idp[k], 0) * page_bytes + poff[k]));
    };
    auto half_to_lds = [&](int i, int k, int half) KV_AI {
      const u32 to = half ? dst[k] ^ 16 : dst[k];
      lds_put(to + i % STAGES * ROOM * 16, to_half8(st[k][2 * half], st[k][2 * half + 1]));
    };
    auto k_frag = [&](int stage, int kb, int ks) KV_AI {
      return sk[stage * ROOM + 32 * kb * (HD / 8) + k_piece<HD>(m32, 2 * ks + hf)];
    };
    auto v_frag = [&](int stage, int db, int g) KV_AI {
      return sv[stage * ROOM + 32 * db * 8 + v_piece(m32, 2 * g + hf)];
    };
    // products 0 .. 4 DB - 1 are those of a tile's weights with its values, the rest the next tile's scores
    constexpr int NV = 4 * DB, NP = NV + 2 * KS, PRE = HD == 64 ? 4 : 6;
    auto frag = [&](int S, int k) KV_AI {
      return k < NV ? v_frag(S % STAGES, k % DB, k / DB) : k_frag((S + 1) % STAGES, (k - NV) & 1, (k - NV) >> 1);
    };
    auto product = [&](int k, h8v f) KV_AI {
      if (k < NV) {
        o[k % DB] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f, p[k / DB], o[k % DB], 0, 0, 0);
      } else {
        const int kb = (k - NV) & 1, ks = (k - NV) >> 1;
        if (ks == 0)
#pragma unroll
          for (int e = 0; e < 16; e++) s[kb][e] = 0.0f;
        s[kb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f, q[ks], s[kb], 0, 0, 0);
      }
    };

    // steps 0 and 1 are staged here (four waves: of the values step 0), the next one's bytes are on their way
    u4v st0[PER], st1[PER];
    lds_barrier();
    if (busy) {
#pragma unroll
      for (int i = 0; i < 3; i++)
#pragma unroll
        for (int k = 0; k < PER; k++) {
          load_id(i, k), load_piece(i, k);
          if (i == 0) st0[k] = st[k];
          if (i == 1) st1[k] = st[k];
        }
    }
    if (wave == 0) load_scales(next);
    {
      v8 w[KS];
      u32 top = 0;
#pragma unroll
      for (int s = 0; s < KS; s++) {
        w[s] = *reinterpret_cast<const v8*>(qp + 16 * s + 8 * hf);
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const u32 bits = __float_as_uint((float)w[s][i]) & 0x7fffffffu;
          top = bits > top ? bits : top;
        }
      }
      const u32 other = (u32)__shfl_xor((int)top, 32, 64);
      top = other > top ? other : top;
      const int e = q_shift(top);
      A = __builtin_amdgcn_ldexpf(a.c, -e);
#pragma unroll
      for (int s = 0; s < KS; s++) q[s] = scaled_q<T>(w[s], e);
    }
    if (busy) {
#pragma unroll
      for (int k = 0; k < PER; k++) {
        const u4v st2 = st[k];
        const bool one = !TURNS && of_values(k);
        st[k] = st0[k], half_to_lds(0, k, 0), half_to_lds(0, k, 1);
        if (!one) st[k] = st1[k], half_to_lds(1, k, 0), half_to_lds(1, k, 1);
        st[k] = one ? st1[k] : st2;
        load_id(one ? 2 : 3, k);
      }
    }
    if (wave == 0) put_granule(0, next);
    lds_barrier();

    // A step: a tile's weights; then its product with V, and the next tile's scores.
    auto step = [&](int i, auto slot_) KV_AI {
      constexpr int S = decltype(slot_)::value;
      if (wave == 0) {
        if (S == 0 && i % 16 == 0) load_page(i + 16, next);
        if (S == 0 && i % 16 == 4) load_scales(next);
        if (S == 0 && i % 16 == 8) put_granule(i + 8, next);
      }
      const int key0 = sp.tile(t0 + i) * 64;
      softmax_tile<DB>(a, s, A, pos, all_seen(a, of_wave, key0, 64), key0 + 8 * hf, meta[i & 31], o, mr, l, p);
      __builtin_amdgcn_sched_barrier(0);
      lds_barrier();
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_setprio(1);
      h8v f[PRE];
#pragma unroll
      for (int k = 0; k < PRE; k++) f[k] = frag(S, k);
      __builtin_amdgcn_sched_barrier(0);
      // Between the products, a part at a time: step i + 2's pieces into LDS, step i + 3's loads, the pages for the
      // loads after those (four waves: of the values each a step nearer). What is past the last tile is for nothing.
      constexpr int PARTS = 3 * PER + 1;
#pragma unroll
      for (int k = 0; k < NP; k++) {
        product(k, f[k % PRE]);
        if (k + PRE < NP) f[k % PRE] = frag(S, k + PRE);
        if (busy)
#pragma unroll
          for (int j = 0; j < PARTS; j++)
            if (k == (2 * j + 1) * NP / (2 * PARTS + 2)) {
              if (j == PARTS - 1) {
#pragma unroll
                for (int c = 0; c < PER; c++) load_id(!TURNS && of_values(c) ? i + 3 : i + 4, c);
              } else {
                const int nearer = !TURNS && of_values(j / 3);
                if (j % 3 == 2) load_piece(i + 3 - nearer, j / 3);
                else half_to_lds(S + 2 - nearer, j / 3, j % 3);
              }
            }
        __builtin_amdgcn_sched_barrier(0);
      }
      __builtin_amdgcn_s_setprio(0);
      __builtin_amdgcn_sched_barrier(0);
      lds_barrier();
      __builtin_amdgcn_sched_barrier(0);
    };
    // The two waves of a SIMD take turns: while one is at its weights the other is at its products.
    if (TURNS && wave >= 4) lds_barrier();
#pragma unroll
    for (int k = NV; k < NP; k++) product(k, frag(STAGES - 1, k));
    lds_barrier();
    for (int i = 0; i < n; i += 4) {
      step(i, std::integral_constant<int, 0>{});
      if (i + 1 < n) step(i + 1, std::integral_constant<int, 1>{});
      if (i + 2 < n) step(i + 2, std::integral_constant<int, 2>{});
      if (i + 3 < n) step(i + 3, std::integral_constant<int, 3>{});
    }
    if (TURNS && wave < 4) lds_barrier();
  }
  l += __shfl_xor(l, 32, 64);
  const long row = mine.row(a);
  if (row < 0) return;
#pragma unroll
  for (int db = 0; db < DB; db++)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const float y[4] = {o[db][i], o[db][i + 1], o[db][i + 2], o[db][i + 3]};
      put<HD, 4, T>(a, row, split, 32 * db + 2 * i + 4 * hf, y, mr, l);
    }
}

// The splits' parts of a row: o = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s. Few parts: hd / 4 lanes a row, its
// parts in turn. Many: a workgroup a row, its groups of hd / 4 lanes every GROUPS-th part each, joined in LDS.
template <int HD, bool MANY, class T>
__global__ __launch_bounds__(256) void kv_attend_join_kernel(AttendArgs a, long row_base, long row_end) {
  constexpr int LPR = HD / 4, GROUPS = 256 / LPR;
  __shared__ f32x4 so[GROUPS][LPR];
  __shared__ float sl[GROUPS];
  const int tid = threadIdx.x, c = tid % LPR, grp = tid / LPR;
  const long R = (long)a.rows.T * a.H, row = row_base + (MANY ? (long)blockIdx.x : (long)blockIdx.x * GROUPS + grp);
  if (!MANY && row >= row_end) return;
  float m = KV_LOWEST;
  if constexpr (MANY) {  // every wave looks at all parts' maxima, a lane each
    for (int s = tid & 63; s < a.splits; s += 64) m = fmaxf(m, a.ml[s * R + row].x);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
  } else {
    for (int s = 0; s < a.splits; s++) m = fmaxf(m, a.ml[s * R + row].x);
  }
  f32x4 o{0, 0, 0, 0};
  float l = 0.0f;
#pragma unroll 4
  for (int s = MANY ? grp : 0; s < a.splits; s += MANY ? GROUPS : 1) {
    const float2 v = a.ml[s * R + row];
    const float f = __builtin_amdgcn_exp2f(v.x - m);
    l = __builtin_fmaf(v.y, f, l);
    o += *reinterpret_cast<const f32x4*>(a.po + (s * R + row) * HD + 4 * c) * f;
  }
  if constexpr (MANY) {
    so[grp][c] = o;
    if (c == 0) sl[grp] = l;
    __syncthreads();
    if (tid >= LPR) return;
    l = 0.0f, o = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < GROUPS; i++) l += sl[i], o += so[i][c];
  }
  const float r = l == 0.0f ? 0.0f : 1.0f / l;
  float y[4] = {o[0] * r, o[1] * r, o[2] * r, o[3] * r};
  store_row<T, 4>(static_cast<T*>(a.o) + row * HD + 4 * c, y);
}

// ------------------------------------------------------------------ the split of a call
enum { KV_FEW1, KV_FEW2, KV_MANY4, KV_MANY8 };  // few rows: 16, 32 to a tile; many rows: four waves, eight
struct Plan {
  int form, m;      // the kernel, and the rows of one of its tiles
  long units;       // bound on the tiles of rows
  int splits, tps;  // splits of the keys, tiles of 64 keys of one
  uint64_t o_bytes, bytes;
};

Plan plan_of(int T, int B, bool packed, int H, int Hkv, int hd, int max_new, int max_len, int window, int sinks) {
  Plan p;
  const int G = H / Hkv;
  const long cus = uwc_cu_count(), rows = (long)(packed ? (max_new > 0 && max_new < T ? max_new : T) : 1) * G;
  const long keys_all = max_len > 0 ? max_len : 1;
  long keys = keys_all;
  if (window && (long)window + sinks + rows / G + 64 < keys) keys = (long)window + sinks + rows / G + 64;
  const long tiles = (keys + 63) / 64;
  // Tiles of 16 rows while at most 80 of them per CU meet a tile of 64 keys (40 of more than 128 rows): they spread best,
  // and the caches serve a key's second reader. Beyond that up to 32 rows still go so (us, 16 rows / many: 5 tokens of 64 heads to 8
  // kv heads, 8 sequences of 20000 136 / 113, 1 of 50000 43 / 45; 16 of 32 heads over 3000, 4 sequences 22 / 29, over
  // 8000, 16 sequences 122 / 98), two tiles of 16 to a wave for heads of 64 and fewer, whose keys cost less to read
  // than to convert (300 tokens of 16 heads, 600 rows, 10 / 16, 1000 of them 50 / 33; 5 tokens of 7 heads to a kv head of 64, 8 x 20000: 92 -> 67, many 74; heads of 128: 78.6 / 78.2).
  const bool light = (rows + 15) / 16 * B * Hkv * tiles <= (rows <= 128 ? 80 : 40) * cus;
  // Many: heads of 128 may take 256 rows to a tile, which share its conversion (4096 tokens over 32768, 2 heads to a kv
  // head, 985 us, 128 rows 1070). 128 rows leave less idle where tiles differ much in length and do not fill
  // the CUs (a prompt of 2000, 4 heads to a kv head, 256 / 128 rows 62 / 56; 512 tokens over 8000 88 / 93, over
  // 30000 256 / 280), where a short window leaves more of a tile's keys to few of 256 rows (8000 tokens, windows of 1000 183 / 178, 2000
  // 292 / 291, 4000 412 / 438), and where sequences have fewer rows than that (16 of up to 100 tokens 187 / 171).
  const bool filled = (long)T * G / 256 * Hkv >= cus;
  const bool wide = hd == 128 && (long)T * G >= 256L * B && (filled ? !window || window >= 2048 : keys_all * G >= 3 * rows);
  p.form = light || rows <= 16 ? KV_FEW1 : hd <= 64 && rows <= 48 ? KV_FEW2 : rows <= 32 ? KV_FEW1 : wide ? KV_MANY8 : KV_MANY4;
  p.m = p.form == KV_FEW1 ? 16 : p.form == KV_FEW2 ? 32 : p.form == KV_MANY4 ? 128 : 256;
  const int M = p.m;
  p.units = packed ? ((long)T * G + M - 1) / M + B : (long)B * ((G + M - 1) / M);
  // Two workgroups of four waves fit a CU. Where rows and heads alone fill the CUs with few-row tiles, their lengths may differ and the
  // keys are cut into pieces that make four rounds' worth (48 sequences of 1500 to 12000 tokens, 8 kv heads: 146 us;
  // two per CU 204, none cut 166); where they do not, into as many as fit at once (one of 131072: 55 us with one or two
  // per CU, 59 with four, 68 with eight), down to one tile a wave (one of 2500: 9.7 us; two tiles 11.8, four 15.6).
  long likely = (long)B * ((rows + M - 1) / M);
  likely = likely < 1 ? 1 : likely < p.units ? likely : p.units;
  const long wgs = likely * Hkv;
  // Many rows: what a split saves in steps of about 1.5 us against what the join costs, a launch and its parts' bytes
  // (1000 tokens of 16 heads over 4000: 66 us in four, 75 in two, 118 in one; 2 x 1000 over none, heads of 64, 22 in one,
  // 30 in two).
  long splits = 1;
  if (p.form <= KV_FEW2) {
    const bool full = wgs >= cus;
    splits = full ? (4 * cus + wgs - 1) / wgs : 2 * cus / wgs;
    const long most = (tiles + (full ? 7 : 3)) / (full ? 8 : 4);
    if (splits > most) splits = most;
    if (splits < 1) splits = 1;
  } else {
    double best = 1e30;
    const long fit = (p.form == KV_MANY8 ? 1 : 2) * cus / wgs;  // eight waves fill a CU
    for (long s = 1; s == 1 || (s <= fit && s <= (tiles + 7) / 8); s++) {
      const double us = 1.5 * ((tiles + s - 1) / s) + (s > 1 ? 7.0 + (double)s * T * H * hd * 8 / 4.8e6 : 0.0);
      if (us < best) best = us, splits = s;
      else if (s > 2 * splits + 8) break;  // past the least
    }
  }
  p.tps = (int)((tiles + splits - 1) / splits);
  p.splits = (int)((tiles + p.tps - 1) / p.tps);
  p.o_bytes = p.splits > 1 ? (uint64_t)p.splits * T * H * hd * 4 : 0;
  p.bytes = p.splits > 1 ? p.o_bytes + (uint64_t)p.splits * T * H * 8 : 0;
  return p;
}

template <int HD, class T>
bool launch_typed(const Plan& p, const AttendArgs& a, dim3 grid, hipStream_t stream) {
  if (p.form == KV_FEW1) {
    hipLaunchKernelGGL((kv_attend_few_kernel<HD, 1, T>), grid, dim3(256), 0, stream, a);
    return true;
  }
  if (p.form == KV_MANY4) {
    hipLaunchKernelGGL((kv_attend_many_kernel<HD, 4, T>), grid, dim3(256), 0, stream, a);
    return true;
  }
  if constexpr (HD <= 64) {
    if (p.form == KV_FEW2) {
      hipLaunchKernelGGL((kv_attend_few_kernel<HD, 2, T>), grid, dim3(256), 0, stream, a);
      return true;
    }
  } else {
    if (p.form == KV_MANY8) {
      hipLaunchKernelGGL((kv_attend_many_kernel<HD, 8, T>), grid, dim3(512), 0, stream, a);
      return true;
    }
  }
  return false;  // the heads have no such form
}
template <int HD>
bool launch(const Plan& p, const AttendArgs& a, int dtype, dim3 grid, hipStream_t stream) {
  return dtype == UWC_KV_BF16 ? launch_typed<HD, __bf16>(p, a, grid, stream) : launch_typed<HD, _Float16>(p, a, grid, stream);
}

}  // namespace

extern "C" uint64_t uwc_kv_attend_scratch_bytes(int T, int B, int packed, int H, int Hkv, int hd, int max_new, int max_len,
                                                int window, int sinks) {
  if (T <= 0 || B < 0 || H <= 0 || Hkv <= 0 || H % Hkv || hd <= 0 || window < 0 || sinks < 0) return 0;
  window = window < 1 << 30 ? window : 1 << 30, sinks = sinks < 1 << 30 ? sinks : 1 << 30;
  return plan_of(T, B, packed != 0, H, Hkv, hd, max_new, max_len, window, sinks).bytes;
}

extern "C" int uwc_kv_attend(const int8_t* k, const int8_t* v, const float* ks, const float* vs, int64_t pages, int page, int Hkv,
                             int hd, const void* q, int64_t q_stride, int dtype, int T, int H, const int32_t* table,
                             int64_t table_stride, int width, const int32_t* lens, const int32_t* cu, int B, int max_new,
                             int max_len, int window, int sinks, float scale, void* scratch, uint64_t scratch_bytes, void* o,
                             hipStream_t stream) {
  const char* fn = "uwc_kv_attend";
  if (!k || !v || !ks || !vs) return uwc_fail("%s: null cache", fn);
  if (pages <= 0 || pages > 0x7fffffff || Hkv <= 0 || Hkv > 65535) return uwc_fail("%s: bad pages=%ld Hkv=%d", fn, (long)pages, Hkv);
  if (page != 16 && page != 32 && page != 64 && page != 128) return uwc_fail("%s: page %d not in {16, 32, 64, 128}", fn, page);
  if (hd != 32 && hd != 64 && hd != 128) return uwc_fail("%s: head_dim %d not in {32, 64, 128}", fn, hd);
  if (dtype != UWC_KV_BF16 && dtype != UWC_KV_FP16) return uwc_fail("%s: unknown dtype %d", fn, dtype);
  if (H <= 0 || H % Hkv) return uwc_fail("%s: H=%d is no multiple of Hkv=%d", fn, H, Hkv);
  if (T < 0 || B < 0 || width < 0 || table_stride < 0) return uwc_fail("%s: bad T=%d B=%d width=%d", fn, T, B, width);
  // positions stay far below 2^30: what is larger is as good as that
  window = window < 1 << 30 ? window : 1 << 30, sinks = sinks < 1 << 30 ? sinks : 1 << 30;
  if (!(scale > 0.0f) || scale > 3e38f) return uwc_fail("%s: the scale of the scores must be positive", fn);
  if (window < 0 || sinks < 0 || (sinks && !window)) return uwc_fail("%s: bad window=%d sinks=%d", fn, window, sinks);
  if (T == 0) return UWC_OK;
  if (!q || !o || (B && (!table || !lens))) return uwc_fail("%s: null arguments", fn);
  if (!cu && T != B) return uwc_fail("%s: without cu every sequence has one row (T=%d B=%d)", fn, T, B);
  if (q_stride % 8 || (((uintptr_t)q | (uintptr_t)o | (uintptr_t)k | (uintptr_t)v | (uintptr_t)scratch) & 15))
    return uwc_fail("%s: q, o, k, v and scratch must be 16-byte aligned", fn);
  if ((int64_t)T * (H / Hkv) > 0x7fffffff - 4096) return uwc_fail("%s: too many rows (T=%d H=%d)", fn, T, H);
  const Plan p = plan_of(T, B, cu != nullptr, H, Hkv, hd, max_new, max_len, window, sinks);
  if (p.bytes && (!scratch || scratch_bytes < p.bytes))
    return uwc_fail("%s: scratch holds %llu bytes, %llu needed", fn, (unsigned long long)(scratch ? scratch_bytes : 0),
                    (unsigned long long)p.bytes);
  const long blocks = p.units * p.splits * Hkv;
  if (blocks * (p.form == KV_MANY8 ? 512 : 256) > 0xFFFFFFFF) return uwc_fail("%s: too many tokens (%d) and heads (%d)", fn, T, H);
  AttendArgs a{k, v, ks, vs, pages, q, q_stride, table, table_stride, width, lens, {cu, B, T}, H, Hkv, H / Hkv,
               __builtin_ctz((unsigned)page), window, sinks, scale * 1.4426950408889634f, (int)p.units, p.splits, p.tps, blocks <= 2L * uwc_cu_count(), o,
               static_cast<float*>(scratch), reinterpret_cast<float2*>(static_cast<char*>(scratch) + p.o_bytes)};
  const dim3 grid((unsigned)blocks), wg(256);
  const bool launched = hd == 32 ? launch<32>(p, a, dtype, grid, stream) : hd == 64 ? launch<64>(p, a, dtype, grid, stream)
                                                                                    : launch<128>(p, a, dtype, grid, stream);
  if (!launched) return uwc_fail("%s: no kernel of form %d for heads of %d", fn, p.form, hd);
  if (int st = uwc_launch_status(fn)) return st;
  if (p.splits == 1) return UWC_OK;
  const long R = (long)T * H;
  const bool many = p.splits > 8;
  const long per = many ? 1 : 1024 / hd;  // rows of a workgroup
#define KV_JOIN(HD)                                                                                                \
  return uwc_launch_rows(fn, (int)((R + per - 1) / per), 256, [&](long g0, int n) {                                \
    const dim3 jg((unsigned)n);                                                                                    \
    const bool bf = dtype == UWC_KV_BF16;                                                                          \
    if (many && bf) hipLaunchKernelGGL((kv_attend_join_kernel<HD, true, __bf16>), jg, wg, 0, stream, a, g0, R);    \
    else if (many) hipLaunchKernelGGL((kv_attend_join_kernel<HD, true, _Float16>), jg, wg, 0, stream, a, g0, R);   \
    else if (bf) hipLaunchKernelGGL((kv_attend_join_kernel<HD, false, __bf16>), jg, wg, 0, stream, a, g0 * per, R); \
    else hipLaunchKernelGGL((kv_attend_join_kernel<HD, false, _Float16>), jg, wg, 0, stream, a, g0 * per, R);      \
  })
  if (hd == 32) KV_JOIN(32);
  if (hd == 64) KV_JOIN(64);
  KV_JOIN(128);
}
