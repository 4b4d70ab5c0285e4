// Linears with 4-bit weights for many rows: both operands through LDS, the weights converted on their way from there to
// the matrix instructions (a conversion of two takes 4 cycles beside the 32 of a product of 32 x 32 x 16, of which two share it).
//
// 8192 x 4096 x 14336 in 706 to 780 us by box (1230 to 1360 TFLOP/s, 82% of the library's bf16 product of the same size), the matrix units busy
// 74% of the cycles (54% of those that the full clock would have); 2048 x 2 x 14336 x 4096, gated, in 397 to 431; 333 x 4096 x 4096 in 24, where few tiles and a barrier a step bound it.
#include "uwc_w4.h"

namespace {

// A workgroup of WM x WN waves makes 64 WM rows of x times 32 NT WN weight rows (where GATED half of a wave's tiles are gate
// rows and the other half the matching up rows), a wave 64 x 32 NT of them on 32 x 32 x 16 instructions. A step is 64 k, two
// groups: lane (i = lane % 32, h = lane / 32) holds weight row i's group h, 32 codes in 16 bytes with one scale, and x's
// values of that group; instruction t multiplies elements 8 t .. 8 t + 7 of both groups.
// Both operands come through LDS, read from memory in whole lines: x by steps, the codes and scales by four steps (128 bytes of a
// row), a quarter of the rows in each step. Each has two buffers. LDS rows are 128 bytes, their 16-byte chunk c at
// c ^ (row / 2 % 8): sixteen lanes that read one chunk of successive rows then touch all 64 banks. Codes straight from
// memory, 32 bytes of each row at a time and by every wave that needs them, kept the address units busier than the matrix units.
// Where tiles of 256 x 256 leave compute units idle, smaller ones, and KG groups of waves that take every KG-th four steps of
// the sums, each with its own buffers; they are added up through LDS, in the groups' order.
template <class T, int KG, int WM, int WN, int NT, bool GATED>
__global__ __launch_bounds__(64 * KG * WM * WN) void w4_gemm_kernel(W4Args a, int mb, int nb) {
  typedef typename W4<T>::v8 v8;
  constexpr int WAVES = WM * WN, BM = 64 * WM, THREADS = 64 * WAVES;  // of a group
  constexpr int ROWS = 32 * NT * WN, BN = GATED ? ROWS / 2 : ROWS;   // of weights, outputs
  // the matching gate and up rows: tiles of one wave, or (one tile a wave) the first and second half of the waves
  constexpr bool PAIRED = GATED && NT > 1;
  constexpr int OT = PAIRED ? NT / 2 : NT;
  constexpr int CHUNKS = BM * 8 / THREADS, PIECE = ROWS * 8 / 4 / THREADS;
  static_assert(PIECE == 1 && ROWS * 2 == THREADS, "a thread stages 16 bytes of codes and one scale a step");
  struct Buffers {
    u8 x[2][BM * 128], codes[2][ROWS * 128], scales[2][ROWS * 8];
  };
  constexpr int SUMS = KG > 1 ? KG * WAVES * NT * 8192 : 0;
  __shared__ __attribute__((aligned(16))) u8 shared[sizeof(Buffers) * KG > SUMS ? sizeof(Buffers) * KG : SUMS];
  const int kg = KG > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / THREADS) : 0, tid = threadIdx.x % THREADS;
  Buffers& L = reinterpret_cast<Buffers*>(shared)[kg];
  const int lane = tid & 63, wave = tid >> 6, wm = wave / WN, wn = wave % WN, i = lane & 31, h = lane >> 5;
  // an XCD takes neighbouring tiles, eight of x's to one of the weight's: its L2 holds what they share
  const int per = (mb * nb + 7) / 8;
  const int tile = blockIdx.x % 8 * per + blockIdx.x / 8;
  if (tile >= mb * nb) return;
  const int band = tile / (8 * nb), rows_in = mb - 8 * band < 8 ? mb - 8 * band : 8, in = tile - band * 8 * nb;
  const int m0 = (8 * band + in % rows_in) * BM, n0 = in / rows_in * BN;
  const int groups = a.K / 32, steps = (groups + 1) / 2;

  // row r of the workgroup's weight rows: tile r / 32, of wave column r / (32 NT); rows past the last are the last, and not stored
  auto weight_row = [&](int r) W4_AI {
    const int t = r / 32 % NT;
    const bool up = PAIRED ? t >= OT : GATED && r >= BN;
    const int n = n0 + (PAIRED ? (r / (32 * NT) * OT + t % OT) * 32 + r % 32 : GATED ? r % BN : r);
    return (long)(n < a.F ? n : a.F - 1) + (up ? a.F : 0);
  };
  const u8* x_at = static_cast<const u8*>(a.x) + (long)m0 * a.x_stride * 2;
  u32 x_off[CHUNKS], to[CHUNKS], from[2], code_from[NT];
  const int chunk = tid & 7;
#pragma unroll
  for (int c = 0; c < CHUNKS; c++) {
    const int r = (tid >> 3) + c * (THREADS / 8), m = m0 + r < a.M ? r : a.M - 1 - m0;
    x_off[c] = (u32)m * (u32)a.x_stride * 2;
    to[c] = r * 128 + ((chunk ^ (r >> 1)) & 7) * 16;
  }
#pragma unroll
  for (int q = 0; q < 2; q++) {  // x rows i and 32 + i of this wave, chunk 4 h
    const int r = wm * 64 + 32 * q + i;
    from[q] = r * 128 + (((4 * h) ^ (r >> 1)) & 7) * 16;
  }
#pragma unroll
  for (int t = 0; t < NT; t++) {  // weight row i of each tile, chunk h
    const int r = (wn * NT + t) * 32 + i;
    code_from[t] = r * 128 + ((h ^ (r >> 1)) & 7) * 16;
  }
  // this thread's weight rows: of piece j of the codes, and of the scales
  const u8* code_at[4];
#pragma unroll
  for (int j = 0; j < 4; j++) code_at[j] = a.codes + weight_row(j * (ROWS / 4) + (tid >> 3)) * (a.K / 2);
  const u8* scale_at = a.scales + weight_row(tid >> 1) * groups;

  w4_u4 xr[CHUNKS], piece;
  u32 scale_byte;
  auto load_x = [&](int s) W4_AI {  // steps past the last are the last; a step's second group may not be there: the first again
    s = s < steps ? s : steps - 1;
    const u32 at = 2 * s + 1 < groups ? chunk * 16 : (chunk & 3) * 16;
#pragma unroll
    for (int c = 0; c < CHUNKS; c++) xr[c] = *reinterpret_cast<const w4_u4*>(x_at + (long)s * 128 + (x_off[c] + at));
  };
  auto put_x = [&](int s) W4_AI {
    if (2 * s + 1 >= groups && (chunk >= 4 || 2 * s >= groups)) {
#pragma unroll
      for (int c = 0; c < CHUNKS; c++) xr[c] = w4_u4{0, 0, 0, 0};
    }
#pragma unroll
    for (int c = 0; c < CHUNKS; c++) *reinterpret_cast<w4_u4*>(&L.x[s & 1][to[c]]) = xr[c];
  };
  // piece j of four steps: of their eight groups, from `first` on, the codes of the j-th quarter of the rows, and bytes j and 4 + j of
  // every row's scales; groups past the last are the last, and meet zeros of x
  auto load_piece = [&](int first, int j, w4_u4& piece, u32& scale_byte) W4_AI {
    const int g = first + chunk, e = first + 4 * (tid & 1) + j;
    piece = *reinterpret_cast<const w4_u4*>(code_at[j] + (g < groups ? g : groups - 1) * 16);
    scale_byte = scale_at[e < groups ? e : groups - 1];
  };
  auto put_piece = [&](int buf, int j, const w4_u4& piece, u32 scale_byte) W4_AI {
    const int r = j * (ROWS / 4) + (tid >> 3);
    *reinterpret_cast<w4_u4*>(&L.codes[buf][r * 128 + ((chunk ^ (r >> 1)) & 7) * 16]) = piece;
    L.scales[buf][(tid >> 1) * 8 + 4 * (tid & 1) + j] = (u8)scale_byte;
  };
  w4_f16 acc[2][NT];
#pragma unroll
  for (int q = 0; q < 2; q++)
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
      for (int r = 0; r < 16; r++) acc[q][t][r] = 0;

  // Loads never depend on a branch, so that the compiler waits for those it needs and no more: the last steps load the
  // last one again.
  {
    w4_u4 first[4];
    u32 bytes[4];
#pragma unroll
    for (int j = 0; j < 4; j++) load_piece(8 * kg, j, first[j], bytes[j]);
    load_x(4 * kg);
    load_piece(8 * (kg + KG), 0, piece, scale_byte);
    __builtin_amdgcn_sched_barrier(0);  // all on their way at once
#pragma unroll
    for (int j = 0; j < 4; j++) put_piece(0, j, first[j], bytes[j]);
    put_x(4 * kg);
    load_x(4 * kg + 1);
  }
  __syncthreads();
  int S = kg;
  for (int four = 0; 4 * (S - kg) < steps; S += KG, four ^= 1) {  // of several groups all go on to the end, with zeros of x
    u2v scale[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
      scale[t] = *reinterpret_cast<const u2v*>(&L.scales[four][((wn * NT + t) * 32 + i) * 8]);
      scale[t][0] >>= 8 * h, scale[t][1] >>= 8 * h;
    }
#pragma unroll
    for (int j = 0; j < 4; j++) {
      if (KG == 1 && 4 * S + j >= steps) break;
      const u8* buf = L.x[j & 1];
      v8 x[2][2];
      w4_u4 codes[NT];
      auto read_x = [&](int t) W4_AI {
#pragma unroll
        for (int q = 0; q < 2; q++) x[t & 1][q] = *reinterpret_cast<const v8*>(buf + (from[q] ^ (t * 16)));
      };
      read_x(0);
#pragma unroll
      for (int t = 0; t < NT; t++) codes[t] = *reinterpret_cast<const w4_u4*>(&L.codes[four][code_from[t] ^ (j * 32)]);
      // what the next step, or the next four, will read has had a whole step to arrive; its place was last read before a barrier
      put_x(j < 3 ? 4 * S + j + 1 : 4 * (S + KG));
      put_piece(four ^ 1, j, piece, scale_byte);
      load_x(j < 2 ? 4 * S + j + 2 : 4 * (S + KG) + j - 2);
      load_piece(8 * (j < 3 ? S + KG : S + 2 * KG), (j + 1) & 3, piece, scale_byte);
      __builtin_amdgcn_sched_barrier(0);  // on their way now, not where the registers are short
#pragma unroll
      for (int t = 0; t < 4; t++) {
        if (t < 3) {
          read_x(t + 1);
          __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int n = 0; n < NT; n++) {
          const u32 f = (scale[n][j >> 1] >> (16 * (j & 1)) & 0xff) << 23;
          const v8 w = W4<T>::weights(codes[n][t], __uint_as_float(f));
#pragma unroll
          for (int q = 0; q < 2; q++) acc[q][n] = W4<T>::mul32(w, x[t & 1][q], acc[q][n]);
        }
      }
      __syncthreads();
    }
  }
  if constexpr (KG > 1) {  // add up: every wave's sums in LDS, four outputs of a row to a thread
    f4v* sums = reinterpret_cast<f4v*>(shared);
    auto slot = [&](int g, int w, int q, int t, int r) W4_AI { return ((((g * WAVES + w) * 2 + q) * NT + t) * 4 + r) * 64; };
#pragma unroll
    for (int q = 0; q < 2; q++)
#pragma unroll
      for (int t = 0; t < NT; t++)
#pragma unroll
        for (int r = 0; r < 4; r++)
          sums[slot(kg, wave, q, t, r) + lane] = f4v{acc[q][t][4 * r], acc[q][t][4 * r + 1], acc[q][t][4 * r + 2], acc[q][t][4 * r + 3]};
    __syncthreads();
    auto sum = [&](int at) W4_AI {
      f4v v = sums[at];
#pragma unroll
      for (int g = 1; g < KG; g++) v += sums[at + slot(g, 0, 0, 0, 0)];
      return v;
    };
    constexpr int COLS = GATED && !PAIRED ? WN / 2 : WN;  // of waves with outputs
    for (int e = threadIdx.x; e < WM * COLS * 2 * OT * 256; e += KG * THREADS) {
      const int l = e % 64, r = e / 64 % 4, t = e / 256 % OT, q = e / (256 * OT) % 2, w = e / (512 * OT), col = w % COLS, row = w / COLS;
      f4v v = sum(slot(0, row * WN + col, q, t, r) + l);
      if (GATED) {
        const f4v u = sum((PAIRED ? slot(0, row * WN + col, q, OT + t, r) : slot(0, row * WN + col + COLS, q, t, r)) + l);
#pragma unroll
        for (int c = 0; c < 4; c++) v[c] = w4_silu(v[c]) * u[c];
      }
      const int m = m0 + row * 64 + 32 * q + l % 32, n = n0 + (col * OT + t) * 32 + 8 * r + 4 * (l / 32);
      if (m < a.M && n < a.F) w4_store<T>(a, m, n, v);
    }
    return;
  }
  auto value = [&](int q, int t, int r) W4_AI {
    f4v v = {acc[q][t][4 * r], acc[q][t][4 * r + 1], acc[q][t][4 * r + 2], acc[q][t][4 * r + 3]};
    if (GATED) {
#pragma unroll
      for (int e = 0; e < 4; e++) v[e] = w4_silu(v[e]) * acc[q][(OT + t) % NT][4 * r + e];
    }
    return v;
  };
  const int mw = m0 + wm * 64, nw = n0 + wn * OT * 32;
  if (a.F % 8 || ((uintptr_t)a.y & 15)) {
#pragma unroll
    for (int q = 0; q < 2; q++)
#pragma unroll
      for (int t = 0; t < OT; t++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const int m = mw + 32 * q + i, n = nw + 32 * t + 8 * r + 4 * h;
          if (m < a.M && n < a.F) w4_store<T>(a, m, n, value(q, t, r));
        }
    return;
  }
  // 32 rows of this wave's outputs at a time through its own part of LDS, so that a row's bytes leave together
  typedef T v4 __attribute__((ext_vector_type(4)));
  constexpr int ROW = 64 * OT, PER = ROW / 16;  // bytes, 16-byte chunks of a row
  static_assert(WAVES * 32 * ROW <= (int)sizeof shared, "the waves' parts fit");
  u8* part = shared + wave * 32 * ROW;
#pragma unroll
  for (int q = 0; q < 2; q++) {
#pragma unroll
    for (int t = 0; t < OT; t++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const f4v v = w4_bias<T>(a, nw + 32 * t + 8 * r + 4 * h, value(q, t, r));
        *reinterpret_cast<v4*>(part + i * ROW + (((4 * t + r) ^ i) % PER) * 16 + 8 * h) = v4{(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
      }
#pragma unroll
    for (int e = 0; e < 32 * PER / 64; e++) {
      const int row = (e * 64 + lane) / PER, c = lane % PER, m = mw + 32 * q + row, n = nw + 8 * c;
      const w4_u4 z = *reinterpret_cast<const w4_u4*>(part + row * ROW + ((c ^ row) % PER) * 16);
      if (m < a.M && n < a.F) *reinterpret_cast<w4_u4*>(static_cast<T*>(a.y) + (long)m * a.F + n) = z;
    }
  }
}

template <class T, int KG, int WM, int WN, int NT, bool GATED>
int launch(const char* fn, const W4Args& a, hipStream_t stream) {
  constexpr int BM = 64 * WM, BN = 32 * NT * WN / (GATED ? 2 : 1), THREADS = 64 * KG * WM * WN;
  const long mb = ((long)a.M + BM - 1) / BM, nb = ((long)a.F + BN - 1) / BN, blocks = (mb * nb + 7) / 8 * 8;
  if (blocks > 0x7fffffffL / THREADS) return uwc_fail("%s: too many rows (%d) and outputs (%d)", fn, a.M, a.F);
  hipLaunchKernelGGL((w4_gemm_kernel<T, KG, WM, WN, NT, GATED>), dim3((unsigned)blocks), dim3(THREADS), 0, stream, a, (int)mb, (int)nb);
  return uwc_launch_status(fn);
}

// us of a round of tiles, one to a compute unit: to begin and end, and a step of a group with one tile alone at work and with all units
// (power, L2). Measured over K = 2048 to 14336; calls of 64 to 2048 rows of 4096 weights, K = 4096, take within 10% of what this says:
// 512 rows 78, 52, 36, 26 and 34 us in the forms' order; 1024 79, 55, 42, 52, 64; 2048 86, 64, 86, 100, 125.
struct Form {
  int BM, rows, KG;
  float fixed, alone, full;
};
const Form forms[] = {{256, 256, 1, 6, 1.09f, 1.55f}, {128, 256, 1, 7, 0.69f, 0.95f}, {128, 128, 2, 7, 0.8f, 1.1f}, {64, 128, 2, 6.5f, 0.47f, 0.62f},
                      {64, 64, 4, 4.2f, 0.7f, 0.75f}};

int choose(const W4Args& a, bool gated, float& least) {
  const long cus = uwc_cu_count(), steps = (a.K + 63) / 64;
  int best = 0;
  for (int f = 0; f < 5; f++) {
    const Form& F = forms[f];
    const long out = F.rows / (gated ? 2 : 1), tiles = (((long)a.M + F.BM - 1) / F.BM) * ((a.F + out - 1) / out), rest = tiles % cus;
    const float times = (steps + 4 * F.KG - 1) / (4 * F.KG) * 4;
    const float us = tiles / cus * (F.fixed + times * F.full) + (rest ? F.fixed + times * (F.alone + (F.full - F.alone) * rest / cus) : 0);
    if (!f || us < least) best = f, least = us;
  }
  return best;
}

template <class T, bool GATED>
int run(const char* fn, const W4Args& a, hipStream_t stream) {
  float us;
  switch (choose(a, GATED, us)) {
    case 0: return launch<T, 1, 4, 2, 4, GATED>(fn, a, stream);
    case 1: return launch<T, 1, 2, 4, 2, GATED>(fn, a, stream);
    case 2: return launch<T, 2, 2, 2, 2, GATED>(fn, a, stream);
    case 3: return launch<T, 2, 1, 4, 1, GATED>(fn, a, stream);
    default: return launch<T, 4, 1, 2, 1, GATED>(fn, a, stream);
  }
}

}  // namespace

float w4_gemm_us(const W4Args& a, bool gated) {
  float us;
  choose(a, gated, us);
  return us;
}

int w4_gemm(const char* fn, const W4Args& a, int dtype, bool gated, hipStream_t stream) {
  if (dtype == UWC_W4_BF16) return gated ? run<__bf16, true>(fn, a, stream) : run<__bf16, false>(fn, a, stream);
  return gated ? run<_Float16, true>(fn, a, stream) : run<_Float16, false>(fn, a, stream);
}
