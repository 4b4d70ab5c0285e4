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
// The running maximum m only moves when some row's new maximum exceeds it by 2^8 or more (w then stays below
// 2^9, far inside fp16), so that most tiles neither exchange maxima between lanes nor rescale O.
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
  int units, splits, tps;
  void* o;
  float* po;   // splits x T H x hd: unnormalised outputs, when splits > 1
  float2* ml;  // splits x T H: their m and denominator
};

constexpr float KV_LOWEST = -1e30f;  // m of a row that has seen nothing
constexpr float KV_SLACK = 8.0f;

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
__device__ __forceinline__ Span span_of(const AttendArgs& a, int p_lo, int p_hi) {
  Span s;
  s.p_lo = p_lo, s.p_hi = p_hi;
  s.lo = a.window && p_lo >= a.window ? p_lo - a.window + 1 : 0;
  s.lt = s.lo >> 6;
  const int first = (a.sinks + 63) >> 6;
  s.st = first < s.lt ? first : s.lt;
  s.n = p_hi < 0 ? 0 : s.st + (p_hi >> 6) - s.lt + 1;
  return s;
}
// Does any row see a key of key0 .. key0 + count - 1? Do all rows see all of them?
__device__ __forceinline__ bool any_seen(const AttendArgs& a, const Span& s, int key0, int count) {
  return key0 <= s.p_hi && (key0 + count > s.lo || key0 < a.sinks);
}
__device__ __forceinline__ bool all_seen(const AttendArgs& a, const Span& s, int key0, int count) {
  return key0 + count - 1 <= s.p_lo && (!a.window || key0 > s.p_hi - a.window || key0 + count <= a.sinks);
}
__device__ __forceinline__ bool seen(const AttendArgs& a, int pos, int key) {
  return key <= pos && (!a.window || key > pos - a.window || key < a.sinks);
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
  int b, j;
  if (a.rows.cu) {
    if (!kv_find(u, a.rows.B, [&](int s) KV_AI { return (int)(((long)kv_new(a.rows, s) * a.G + M - 1) / M); }, b, j)) return false;
    x.row0 = a.rows.cu[b];
  } else {
    const int per = (a.G + M - 1) / M;
    b = u / per, j = u % per;
    x.row0 = b;
  }
  x.b = b, x.r0 = j * M, x.rows = kv_new(a.rows, b) * a.G, x.len = a.lens[b];
  return true;
}

// The packed row and head of row r of a unit as an index into (T, H), or -1.
__device__ __forceinline__ long out_row(const AttendArgs& a, const Unit& x, int r, int h) {
  const int t = x.row0 + r / a.G;
  return r < x.rows && t >= 0 && t < a.rows.T ? (long)t * a.H + h * a.G + r % a.G : -1;
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
// each, straight from memory into registers; their results meet in LDS.
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
    const long row = out_row(a, x, r, h);
    pos[rb] = row < 0 ? -1 : x.pos(a, r);
    const T* qp = static_cast<const T*>(a.q) + (row < 0 ? 0 : (row / a.H) * a.q_stride + (row % a.H) * HD);
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
      if (!whole)
#pragma unroll
        for (int i = 0; i < 16; i++) e[i] = seen(a, pos[rb], kt * 64 + 16 * g + i) ? e[i] : -__builtin_inff();
#pragma unroll
      for (int i = 0; i < 16; i++) top = fmaxf(top, e[i]);
      if (__any(top > mr[rb] + KV_SLACK)) {
        const float to = fmaxf(mr[rb], max_xor32(max_xor16(top)));
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
    const long row = out_row(a, x, x.r0 + rr, h);
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

// The splits' parts of one row: o = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s.
template <int HD, class T>
__global__ __launch_bounds__(256) void kv_attend_join_kernel(AttendArgs a, long row_base) {
  constexpr int LPR = HD / 4, GROUPS = 256 / LPR;  // lanes of 4 dims per part; parts read at once
  __shared__ f32x4 so[GROUPS][LPR];
  __shared__ float sl[GROUPS];
  const int tid = threadIdx.x, c = tid % LPR, grp = tid / LPR;
  const long R = (long)a.rows.T * a.H, row = row_base + blockIdx.x;
  float m = KV_LOWEST;
  for (int s = 0; s < a.splits; s++) m = fmaxf(m, a.ml[s * R + row].x);
  f32x4 o{0, 0, 0, 0};
  float l = 0.0f;
  for (int s = grp; s < a.splits; s += GROUPS) {
    const float2 v = a.ml[s * R + row];
    const float f = __builtin_amdgcn_exp2f(v.x - m);
    l = __builtin_fmaf(v.y, f, l);
    o += *reinterpret_cast<const f32x4*>(a.po + (s * R + row) * HD + 4 * c) * f;
  }
  so[grp][c] = o;
  if (c == 0) sl[grp] = l;
  __syncthreads();
  if (tid >= LPR) return;
  l = 0.0f, o = f32x4{0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < GROUPS; i++) l += sl[i], o += so[i][c];
  const float r = l == 0.0f ? 0.0f : 1.0f / l;
  float y[4] = {o[0] * r, o[1] * r, o[2] * r, o[3] * r};
  store_row<T, 4>(static_cast<T*>(a.o) + row * HD + 4 * c, y);
}

// ------------------------------------------------------------------ the split of a call
struct Plan {
  int rb;              // 16-row blocks of a tile of rows
  long units;          // bound on the tiles of rows
  int splits, tps;     // splits of the keys, tiles of 64 keys of one
  uint64_t o_bytes, bytes;
};

Plan plan_of(int T, int B, bool packed, int H, int Hkv, int hd, int max_new, int max_len, int window, int sinks) {
  Plan p;
  const int G = H / Hkv;
  const long rows = (long)(packed ? (max_new > 0 && max_new < T ? max_new : T) : 1) * G;
  (void)rows;
  p.rb = 1;
  const int M = 16 * p.rb;
  p.units = packed ? ((long)T * G + M - 1) / M + B : (long)B * ((G + M - 1) / M);
  long keys = max_len > 0 ? max_len : 1;
  if (window && (long)window + sinks + M / G + 128 < keys) keys = (long)window + sinks + M / G + 128;
  const long tiles = (keys + 63) / 64, want = 2L * uwc_cu_count() / (p.units * Hkv);
  long splits = want < 1 ? 1 : want;
  if (splits > (tiles + 3) / 4) splits = (tiles + 3) / 4;
  if (splits > 1024) splits = 1024;
  p.tps = (int)((tiles + splits - 1) / splits);
  p.splits = (int)((tiles + p.tps - 1) / p.tps);
  p.o_bytes = p.splits > 1 ? (uint64_t)p.splits * T * H * hd * 4 : 0;
  p.bytes = p.splits > 1 ? p.o_bytes + (uint64_t)p.splits * T * H * 8 : 0;
  return p;
}

}  // namespace

extern "C" uint64_t uwc_kv_attend_scratch_bytes(int T, int B, int packed, int H, int Hkv, int hd, int max_new, int max_len,
                                                int window, int sinks) {
  if (T <= 0 || B <= 0 || H <= 0 || Hkv <= 0 || H % Hkv || hd <= 0 || window < 0 || sinks < 0) return 0;
  return plan_of(T, B, packed != 0, H, Hkv, hd, max_new, max_len, window, sinks).bytes;
}

extern "C" int uwc_kv_attend(const int8_t* k, const int8_t* v, const float* ks, const float* vs, int64_t pages, int page, int Hkv,
                             int hd, const void* q, int64_t q_stride, int dtype, int T, int H, const int32_t* table,
                             int64_t table_stride, int width, const int32_t* lens, const int32_t* cu, int B, int max_new,
                             int max_len, int window, int sinks, float scale, void* scratch, uint64_t scratch_bytes, void* o,
                             hipStream_t stream) {
  const char* fn = "uwc_kv_attend";
  if (!k || !v || !ks || !vs) return uwc_fail("%s: null cache", fn);
  if (pages <= 0 || pages > 0x7fffffff || Hkv <= 0) return uwc_fail("%s: bad pages=%ld Hkv=%d", fn, (long)pages, Hkv);
  if (page != 16 && page != 32 && page != 64 && page != 128) return uwc_fail("%s: page %d not in {16, 32, 64, 128}", fn, page);
  if (hd != 32 && hd != 64 && hd != 128) return uwc_fail("%s: head_dim %d not in {32, 64, 128}", fn, hd);
  if (dtype != UWC_KV_BF16 && dtype != UWC_KV_FP16) return uwc_fail("%s: unknown dtype %d", fn, dtype);
  if (H <= 0 || H % Hkv) return uwc_fail("%s: H=%d is no multiple of Hkv=%d", fn, H, Hkv);
  if (T < 0 || B < 0 || width < 0 || table_stride < 0) return uwc_fail("%s: bad T=%d B=%d width=%d", fn, T, B, width);
  if (window < 0 || sinks < 0 || (sinks && !window)) return uwc_fail("%s: bad window=%d sinks=%d", fn, window, sinks);
  if (T == 0 || B == 0) return UWC_OK;
  if (!q || !table || !lens || !o) return uwc_fail("%s: null arguments", fn);
  if (!cu && T != B) return uwc_fail("%s: without cu every sequence has one row (T=%d B=%d)", fn, T, B);
  if (q_stride % 8 || (((uintptr_t)q | (uintptr_t)o | (uintptr_t)k | (uintptr_t)v | (uintptr_t)scratch) & 15))
    return uwc_fail("%s: q, o, k, v and scratch must be 16-byte aligned", fn);
  if ((int64_t)T * (H / Hkv) > 0x7fffffff - 4096) return uwc_fail("%s: too many rows (T=%d H=%d)", fn, T, H);
  const Plan p = plan_of(T, B, cu != nullptr, H, Hkv, hd, max_new, max_len, window, sinks);
  if (p.bytes && (!scratch || scratch_bytes < p.bytes))
    return uwc_fail("%s: scratch holds %llu bytes, %llu needed", fn, (unsigned long long)(scratch ? scratch_bytes : 0),
                    (unsigned long long)p.bytes);
  const long blocks = p.units * p.splits * Hkv;
  if (blocks > 0xFFFFFF) return uwc_fail("%s: too many tokens (%d) and heads (%d)", fn, T, H);  // 2^32 threads
  AttendArgs a{k, v, ks, vs, pages, q, q_stride, table, table_stride, width, lens, {cu, B, T}, H, Hkv, H / Hkv,
               __builtin_ctz((unsigned)page), window, sinks, scale * 1.4426950408889634f, (int)p.units, p.splits, p.tps, o,
               static_cast<float*>(scratch), reinterpret_cast<float2*>(static_cast<char*>(scratch) + p.o_bytes)};
  const dim3 grid((unsigned)blocks), wg(256);
#define KV_FEW(HD)                                                                                              \
  do {                                                                                                          \
    if (dtype == UWC_KV_BF16) hipLaunchKernelGGL((kv_attend_few_kernel<HD, 1, __bf16>), grid, wg, 0, stream, a); \
    else hipLaunchKernelGGL((kv_attend_few_kernel<HD, 1, _Float16>), grid, wg, 0, stream, a);                   \
  } while (0)
  if (hd == 32) KV_FEW(32);
  else if (hd == 64) KV_FEW(64);
  else KV_FEW(128);
  if (int st = uwc_launch_status(fn)) return st;
  if (p.splits == 1) return UWC_OK;
#define KV_JOIN(HD)                                                                                                       \
  return uwc_launch_rows(fn, T * H, 256, [&](long r0, int n) {                                                            \
    if (dtype == UWC_KV_BF16) hipLaunchKernelGGL((kv_attend_join_kernel<HD, __bf16>), dim3((unsigned)n), wg, 0, stream, a, r0); \
    else hipLaunchKernelGGL((kv_attend_join_kernel<HD, _Float16>), dim3((unsigned)n), wg, 0, stream, a, r0);              \
  })
  if (hd == 32) KV_JOIN(32);
  if (hd == 64) KV_JOIN(64);
  KV_JOIN(128);
}
