// Which page of the paged key/value cache (layout in uwc_kv.h) belongs to whom: sequences that branch, end and grow, and
// the pages in use moved to the front.
//
//   fork     row i of the new page table continues old row parents[i]. A page's count goes up by one for each further row
//            that shares it and down by one for each old row that nobody continues; what a row may still write, its
//            last, partly filled page, is its own: the first row of a parent keeps it, the others (and the first too, where
//            the count says that others hold it) get copies. Pages wanted are taken from those with no count, lowest first,
//            row by row.
//   compact  of n pages in use those from n on, in their order, go to the free ones below n.
//
// Two launches each. The first writes one bit a page (free, or in use), sums of them over 1024 pages, and what each row
// needs; the second's workgroups find a page by its rank from those sums, each for itself, copy, and write
// tables and counts. Nothing goes by the order in which workgroups run. Copies are bound by HBM, in pieces of at most 32 KB to a
// workgroup (1.76 GB in 375 us, 4.7 TB/s, what a copy reaches here; one prompt into 32 rows, 171 MB in 32); the rest is a chain of short
// dependent loads (256 rows of 252 entries, nothing copied: 9 + 5 us).
#include "uwc_kv.h"

namespace {

constexpr int RANGE = 1024, WORDS = RANGE / 64;  // pages, words of 64 bits of a range
constexpr int ROWS = 4096, RANGES = 2048;        // most rows and ranges of a call: 32 KB of LDS, four workgroups to a unit
constexpr int LAYERS = 64;                       // layers of a launch
constexpr int UNITS = 2048;                      // 16-byte units of a piece

// What a row of the new table needs: `fresh` pages, for its entries from `first_fresh` on that are not there, the first of them for
// a copy where tail is not -1: of page `tail`, or, where the first row of a parent takes one and gives its own count back, -2 - tail.
struct Row {
  int fresh, tail, granules, first_fresh;
};

struct Scratch {
  u64* bits;
  int* sums;
  Row* rows;
};

struct Layers {
  u8 *k[LAYERS], *v[LAYERS];
  float *ks[LAYERS], *vs[LAYERS];
  int n, Hkv, hd, page;
};

struct ForkArgs {
  const int* table;
  long stride;
  int width;
  const int* lens;
  int B;
  const int* refs;
  int pages;
  const int* parents;
  int R, room, page;
  int *new_table, *new_lens, *new_refs, *missing;
  Scratch s;
};

struct CompactArgs {
  const int* table;
  long stride;
  int width, B;
  const int* refs;
  int pages;
  int *new_table, *new_refs;
  Scratch s;
};

// A number that is the same in all lanes, as a scalar: what it indexes is then no select over all layers.
__device__ __forceinline__ int uniform(long x) { return __builtin_amdgcn_readfirstlane((int)x); }

__device__ __forceinline__ int div_up(int a, int b) { return a / b + (a % b != 0); }

// One wave: the word of pages 64 w .. 64 w + 63 with a bit where `set`; returns how many.
__device__ __forceinline__ int put_word(u64* bits, long w, bool set) {
  const u64 b = __ballot(set);
  if ((threadIdx.x & 63) == 0) bits[w] = b;
  return __builtin_popcountll(b);
}

// The workgroup's exclusive sums of get(0) .. get(n - 1), given to put(i, sum), and the total. 256 threads.
template <class G, class P>
__device__ __forceinline__ int scan(int n, int* tmp, G&& get, P&& put) {
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  int before = 0;
  for (int i0 = 0; i0 < n; i0 += 256) {
    const int v = i0 + t < n ? get(i0 + t) : 0;
    int s = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(s, d, 64);
      if (lane >= d) s += o;
    }
    if (lane == 63) tmp[wave] = s;
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int w = 0; w < 4; w++) {
      if (w < wave) s += tmp[w];
      all += tmp[w];
    }
    if (i0 + t < n) put(i0 + t, before + s - v);
    before += all;
    __syncthreads();
  }
  return before;
}

// Number `rank` of the pages whose bit is `ONE`: in the last range with at most `rank` of them before it.
template <bool ONE>
__device__ __forceinline__ int select(const int* sums, int ranges, const u64* bits, int rank) {
  auto before = [&](int r) KV_AI { return ONE ? sums[r] : r * RANGE - sums[r]; };
  int lo = 0, hi = ranges - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (before(mid) <= rank) lo = mid;
    else hi = mid - 1;
  }
  rank -= before(lo);
#pragma unroll 4
  for (int w = 0; w < WORDS; w++) {
    u64 b = bits[(long)lo * WORDS + w];
    if (!ONE) b = ~b;
    const int c = __builtin_popcountll(b);
    if (rank < c) {
      int at = 0;  // the rank-th set bit, by halves
#pragma unroll
      for (int d = 32; d; d >>= 1) {
        const int low = __builtin_popcountll(b & ((1ull << d) - 1));
        if (rank >= low) rank -= low, at += d, b >>= d;
      }
      return lo * RANGE + w * 64 + at;
    }
    rank -= c;
  }
  return -1;
}

// How many bits are set before page p.
__device__ __forceinline__ int rank_of(const int* sums, const u64* bits, int p) {
  int n = sums[p / RANGE];
  const u64* b = bits + (long)(p / RANGE) * WORDS;
  for (int w = 0; w < p % RANGE / 64; w++) n += __builtin_popcountll(b[w]);
  return p % 64 ? n + __builtin_popcountll(b[p % RANGE / 64] & ((1ull << (p % 64)) - 1)) : n;
}

// Pieces of one page's copy in one layer: keys and values, each in as many as its bytes need.
__device__ __forceinline__ int pieces_of(const Layers& L) { return 2 * div_up(L.Hkv * (L.page / 16) * L.hd, UNITS); }

// Piece `piece` of page src's first `granules` granules to page dst: bytes, and with the first piece of either side its scales.
__device__ __forceinline__ void copy(const Layers& L, int layer, int piece, int src, int dst, int granules) {
  const bool values = piece & 1;
  const long bytes = (long)L.Hkv * L.page * L.hd;
  const u8* from = (values ? L.v[layer] : L.k[layer]) + src * bytes;
  u8* to = (values ? L.v[layer] : L.k[layer]) + dst * bytes;
  const u32 g = granules, of_head = g * L.hd, all = of_head * L.Hkv, whole = L.page / 16;
  if ((piece >> 1) * UNITS >= all) return;
  u4v z[UNITS / 256];
  u32 at[UNITS / 256];
#pragma unroll
  for (int i = 0; i < UNITS / 256; i++) {
    const u32 f = (piece >> 1) * UNITS + i * 256 + threadIdx.x, e = f < all ? f : all - 1;  // what is past the last is read and not stored
    at[i] = g == whole ? e : values ? e / g * whole + e % g : e / of_head * (whole * L.hd) + e % of_head;
    z[i] = *reinterpret_cast<const u4v*>(from + (long)at[i] * 16);
  }
#pragma unroll
  for (int i = 0; i < UNITS / 256; i++)
    if ((piece >> 1) * UNITS + i * 256 + threadIdx.x < all) *reinterpret_cast<u4v*>(to + (long)at[i] * 16) = z[i];
  if (piece < 2) {
    float* s = values ? L.vs[layer] : L.ks[layer];
    for (int h = threadIdx.x; h < L.Hkv; h += 256) s[(long)dst * L.Hkv + h] = s[(long)src * L.Hkv + h];
  }
}

// This workgroup's share of `moves` pages in all layers: find(move) once for each move it works on, then each(layer, piece). Where there
// are fewer moves than workgroups, several share one (a search for each piece took 59 us for 350 small pages in 18 layers).
template <class S, class F>
__device__ __forceinline__ void share(const Layers& L, int moves, S&& find, F&& each) {
  const int pieces = pieces_of(L), per = L.n * pieces, groups = gridDim.x;
  if (!per || !moves) return;
  const int to_a_move = moves >= groups ? 1 : groups / moves < per ? groups / moves : per, at_once = groups / to_a_move;
  const int part = uniform(blockIdx.x % to_a_move);
  int move = uniform(blockIdx.x / to_a_move);
  if (move >= at_once) return;  // what is left over of the workgroups
  for (; move < moves; move += at_once) {
    find(move);
    for (int rest = part; rest < per; rest += to_a_move) each(uniform(rest / pieces), uniform(rest % pieces));
  }
}

// The sums of a range's bits of `get`: 256 threads, a wave to every fourth word.
template <class G>
__device__ __forceinline__ void put_range(const Scratch& s, int range, int pages, int* tmp, G&& get) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int n = 0;
  for (int w = wave; w < WORDS; w += 4) {
    const int p = range * RANGE + w * 64 + lane;
    n += put_word(s.bits, (long)range * WORDS + w, p < pages && get(p));
  }
  if (lane == 0) tmp[wave] = n;
  __syncthreads();
  if (threadIdx.x == 0) s.sums[range] = tmp[0] + tmp[1] + tmp[2] + tmp[3];
}

__global__ __launch_bounds__(256) void fork_plan_kernel(ForkArgs a, int ranges) {
  __shared__ int children[ROWS], change[RANGE], tmp[4], listed;
  __shared__ unsigned short list[ROWS];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  auto length = [&](int r) KV_AI {
    const int n = a.lens[r];
    const long most = (long)a.width * a.page;
    return n < 0 ? 0 : n > most ? (int)most : n;
  };
  if (blockIdx.x < ranges) {  // the counts of a range of pages without what is handed out, and which are free
    const int p0 = blockIdx.x * RANGE;
    for (int r = t; r < a.B; r += 256) children[r] = 0;
    for (int p = t; p < RANGE; p += 256) change[p] = 0;
    __syncthreads();
    for (int i = t; i < a.R; i += 256) {
      const int r = a.parents[i];
      if (r >= 0 && r < a.B) atomicAdd(&children[r], 1);
    }
    __syncthreads();
    // the rows whose pages change hands, in any order: they are added up; then all their entries, eight to a thread on their way
    if (t == 0) listed = 0;
    __syncthreads();
    for (int r = t; r < a.B; r += 256)
      if (children[r] != 1) list[atomicAdd(&listed, 1)] = (unsigned short)r;
    __syncthreads();
    const u32 entries = (u32)listed * a.width;
    for (u32 e0 = t; e0 < entries; e0 += 256 * 8) {
      int p[8], c[8];
#pragma unroll
      for (int k = 0; k < 8; k++) {
        const u32 e = e0 + 256 * k < entries ? e0 + 256 * k : entries - 1, at = e / a.width, j = e % a.width;
        const int r = list[at];
        p[k] = a.table[r * a.stride + j];
        c[k] = children[r] ? (int)j < length(r) / a.page ? children[r] - 1 : 0 : -1;
        if (e0 + 256 * k >= entries) c[k] = 0;
      }
#pragma unroll
      for (int k = 0; k < 8; k++)
        if (c[k] && p[k] >= p0 && p[k] < p0 + RANGE && p[k] < a.pages) atomicAdd(&change[p[k] - p0], c[k]);
    }
    __syncthreads();
    put_range(a.s, blockIdx.x, a.pages, tmp, [&](int p) KV_AI {
      const int n = a.refs[p] + change[p - p0];
      a.new_refs[p] = n;
      return n <= 0;
    });
    return;
  }
  const int i = blockIdx.x - ranges, r = a.parents[i];
  int* out = a.new_table + (long)i * a.width;
  if (r < 0 || r >= a.B) {
    for (int j = t; j < a.width; j += 256) out[j] = -1;
    if (t == 0) a.new_lens[i] = 0, a.s.rows[i] = Row{0, -1, 0, 0};
    return;
  }
  const int* row = a.table + r * a.stride;
  const int n = length(r), full = n / a.page, rest = n % a.page, have = full + (rest != 0);
  const long longer = ((long)n + a.room + a.page - 1) / a.page;
  const int want = longer < a.width ? (int)longer : a.width;
  bool earlier = false;
  for (int e = t; e < i; e += 256) earlier |= a.parents[e] == r;
  const bool first = !__syncthreads_or(earlier);
  const int tail = rest ? row[full] : -1;
  const bool own = tail >= 0 && tail < a.pages, copied = own && (!first || a.refs[tail] > 1);
  int fresh = 0;
  for (int j = t; j < a.width; j += 256) {
    const int p = first || j < full ? row[j] : -1;
    const bool wanted = (copied && j == full) || (p < 0 && j >= have && j < want);
    out[j] = wanted ? -1 : p;
    fresh += wanted;
  }
  if (!first && rest && !own && t == full % 256) out[full] = tail;  // what is not in the cache stays so
#pragma unroll
  for (int d = 32; d; d >>= 1) fresh += __shfl_xor(fresh, d, 64);
  if (lane == 0) tmp[wave] = fresh;
  __syncthreads();
  if (t == 0) {
    a.new_lens[i] = n;
    a.s.rows[i] = Row{tmp[0] + tmp[1] + tmp[2] + tmp[3], copied ? (first ? -2 - tail : tail) : -1, (rest + 15) / 16, copied ? full : have};
  }
}

__global__ __launch_bounds__(256) void fork_finish_kernel(ForkArgs a, Layers L, int ranges, bool first_launch) {
  __shared__ int sums[RANGES], rank[ROWS], tmp[4];
  __shared__ unsigned short copies[ROWS];
  const int t = threadIdx.x;
  const int free = scan(ranges, tmp, [&](int r) KV_AI { return a.s.sums[r]; }, [&](int r, int s) KV_AI { sums[r] = s; });
  const int wanted = scan(a.R, tmp, [&](int i) KV_AI { return a.s.rows[i].fresh; }, [&](int i, int s) KV_AI { rank[i] = s; });
  // the rows whose copy has a page to go to
  const int n = scan(a.R, tmp, [&](int i) KV_AI { return (int)(a.s.rows[i].tail != -1 && rank[i] < free); },
                     [&](int i, int s) KV_AI { if (a.s.rows[i].tail != -1 && rank[i] < free) copies[s] = (unsigned short)i; });
  if (first_launch) {
    if (blockIdx.x == 0 && t == 0) *a.missing = wanted > free ? wanted - free : 0;
    for (int i = blockIdx.x; i < a.R; i += gridDim.x) {
      const Row r = a.s.rows[i];
      if (t == 0 && r.tail < -1) atomicSub(&a.new_refs[-2 - r.tail], 1);
      // the entries that are wanted are those from the first one on that are not there
      int left = r.fresh, at = rank[i];
      for (int j0 = r.first_fresh; left > 0 && j0 < a.width; j0 += 64) {
        const int j = j0 + (t & 63);
        int* e = a.new_table + (long)i * a.width + j;
        const bool open = j < a.width && *e < 0;
        const u64 m = __ballot(open);
        const int mine = __builtin_popcountll(m & ((1ull << (t & 63)) - 1));
        __syncthreads();
        if (t < 64 && open && mine < left && at + mine < free) {
          const int p = select<true>(sums, ranges, a.s.bits, at + mine);
          *e = p;
          a.new_refs[p] = 1;
        }
        __syncthreads();
        const int c = __builtin_popcountll(m);
        at += c, left -= c;
      }
    }
  }
  int src = 0, dst = 0, granules = 0;
  share(L, n, [&](int move) KV_AI {
    const int i = copies[move];
    const Row r = a.s.rows[i];
    src = uniform(r.tail < -1 ? -2 - r.tail : r.tail), granules = uniform(r.granules);
    dst = uniform(select<true>(sums, ranges, a.s.bits, rank[i]));
  }, [&](int layer, int piece) KV_AI { copy(L, layer, piece, src, dst, granules); });
}

__global__ __launch_bounds__(256) void compact_plan_kernel(CompactArgs a) {
  __shared__ int tmp[4];
  put_range(a.s, blockIdx.x, a.pages, tmp, [&](int p) KV_AI { return a.refs[p] > 0; });
}

__global__ __launch_bounds__(256) void compact_finish_kernel(CompactArgs a, Layers L, int ranges, bool first_launch) {
  __shared__ int sums[RANGES], tmp[4];
  const int used = scan(ranges, tmp, [&](int r) KV_AI { return a.s.sums[r]; }, [&](int r, int s) KV_AI { sums[r] = s; });
  const u64* bits = a.s.bits;
  const int kept = used < a.pages ? rank_of(sums, bits, used) : used;  // those below `used` stay
  if (first_launch) {
    auto in_use = [&](int p) KV_AI { return bits[p / 64] >> (p % 64) & 1; };
    auto target = [&](int p) KV_AI { return select<false>(sums, ranges, bits, rank_of(sums, bits, p) - kept); };
    const int me = blockIdx.x * 256 + threadIdx.x, step = gridDim.x * 256;
    for (int p = me; p < a.pages; p += step) {
      if (in_use(p)) a.new_refs[p < used ? p : target(p)] = a.refs[p];
      if (p >= used) a.new_refs[p] = 0;
    }
    for (u32 e = me; e < (u32)a.B * a.width; e += step) {
      const int p = a.table[(long)(e / a.width) * a.stride + e % a.width];
      a.new_table[e] = p >= used && p < a.pages && in_use(p) ? target(p) : p;
    }
  }
  int src = 0, dst = 0;
  share(L, used - kept, [&](int move) KV_AI {
    src = uniform(select<true>(sums, ranges, bits, kept + move)), dst = uniform(select<false>(sums, ranges, bits, move));
  }, [&](int layer, int piece) KV_AI { copy(L, layer, piece, src, dst, L.page / 16); });
}

long ranges_of(long pages) { return (pages + RANGE - 1) / RANGE; }

Scratch cut(void* scratch, long pages, int R) {
  u8* p = static_cast<u8*>(scratch);
  const long bits = ranges_of(pages) * (WORDS * 8);
  return Scratch{reinterpret_cast<u64*>(p), reinterpret_cast<int*>(p + bits + R * sizeof(Row)), reinterpret_cast<Row*>(p + bits)};
}

int check(const char* fn, int layers, void* const* caches, int64_t pages, int page, int Hkv, int hd, const void* table, int64_t stride,
          int width, int B, const void* refs, const void* scratch, uint64_t bytes, int R) {
  if (layers < 0 || (layers && !caches)) return uwc_fail("%s: bad layers=%d", fn, layers);
  if (pages <= 0 || pages > (int64_t)RANGE * RANGES || Hkv <= 0 || Hkv > 65535)
    return uwc_fail("%s: bad pages=%ld (at most %ld) Hkv=%d", fn, (long)pages, (long)RANGE * RANGES, Hkv);
  if (page != 16 && page != 32 && page != 64 && page != 128) return uwc_fail("%s: page %d not in {16, 32, 64, 128}", fn, page);
  if (hd != 32 && hd != 64 && hd != 128) return uwc_fail("%s: head_dim %d not in {32, 64, 128}", fn, hd);
  if (width < 0 || B < 0 || B > ROWS || R < 0 || R > ROWS || stride < 0)
    return uwc_fail("%s: bad width=%d, rows %d and %d (at most %d)", fn, width, B, R, ROWS);
  if ((long)(B > R ? B : R) * width > 0x7fffffff) return uwc_fail("%s: a table of %d rows of %d entries, more than 2^31", fn, B > R ? B : R, width);
  if ((B && width && !table) || !refs || !scratch) return uwc_fail("%s: null arguments", fn);
  if (bytes < uwc_kv_pages_scratch_bytes(pages, R) || ((uintptr_t)scratch & 15)) return uwc_fail("%s: the scratch is too small or not 16-byte aligned", fn);
  for (int i = 0; i < 4 * layers; i++) {
    if (!caches[i]) return uwc_fail("%s: null cache", fn);
    if (i % 4 < 2 && ((uintptr_t)caches[i] & 15)) return uwc_fail("%s: k and v must be 16-byte aligned", fn);
  }
  return UWC_OK;
}

// go(layers of a launch, whether it is the first); one launch without any layers
template <class Go>
int by_layers(const char* fn, int layers, void* const* caches, int Hkv, int hd, int page, Go&& go) {
  for (int l0 = 0; l0 == 0 || l0 < layers; l0 += LAYERS) {
    Layers L;
    L.n = layers - l0 < LAYERS ? layers - l0 : LAYERS, L.Hkv = Hkv, L.hd = hd, L.page = page;
    for (int l = 0; l < L.n; l++) {
      void* const* c = caches + 4 * (l0 + l);
      L.k[l] = static_cast<u8*>(c[0]), L.v[l] = static_cast<u8*>(c[1]), L.ks[l] = static_cast<float*>(c[2]), L.vs[l] = static_cast<float*>(c[3]);
    }
    go(L, l0 == 0);
    if (int st = uwc_launch_status(fn)) return st;
  }
  return UWC_OK;
}

// Workgroups of the second launch: as many as there can be jobs, up to what the compute units hold at once, which then take several
// each (fork: four to a unit; four rounds of them, each finding its rows' ranks, took 10.5 us where nothing is copied).
unsigned grid_of(int to_a_unit, long jobs, long rows) {
  const long most = (long)to_a_unit * uwc_cu_count(), n = jobs > rows ? jobs : rows;
  return (unsigned)(n < 1 ? 1 : n < most ? n : most);
}

long pieces_on_host(int Hkv, int page, int hd) { return 2 * (((long)Hkv * (page / 16) * hd + UNITS - 1) / UNITS); }

}  // namespace

extern "C" uint64_t uwc_kv_pages_scratch_bytes(int64_t pages, int rows) {
  if (pages <= 0 || rows < 0) return 0;
  return (uint64_t)ranges_of(pages) * (WORDS * 8 + 4) + (uint64_t)rows * sizeof(Row);
}

extern "C" int uwc_kv_fork(int layers, void* const* caches, int64_t pages, int page, int Hkv, int hd, const int32_t* table,
                           int64_t table_stride, int width, const int32_t* lens, int B, const int32_t* refs, const int32_t* parents,
                           int R, int room, int32_t* new_table, int32_t* new_lens, int32_t* new_refs, int32_t* missing, void* scratch,
                           uint64_t scratch_bytes, hipStream_t stream) {
  const char* fn = "uwc_kv_fork";
  if (int st = check(fn, layers, caches, pages, page, Hkv, hd, table, table_stride, width, B, refs, scratch, scratch_bytes, R)) return st;
  if (room < 0) return uwc_fail("%s: room=%d", fn, room);
  if ((long)width * page > 0x7fffffff) return uwc_fail("%s: a table row of %d pages holds more than 2^31 tokens", fn, width);
  if ((B && !lens) || (R && (!parents || !new_lens || (width && !new_table))) || !new_refs || !missing) return uwc_fail("%s: null arguments", fn);
  ForkArgs a{table, (long)table_stride, width, lens, B, refs, (int)pages, parents, R, room, page, new_table, new_lens, new_refs, missing,
             cut(scratch, pages, R)};
  const int ranges = (int)ranges_of(pages);
  hipLaunchKernelGGL(fork_plan_kernel, dim3(ranges + R), dim3(256), 0, stream, a, ranges);
  if (int st = uwc_launch_status(fn)) return st;
  return by_layers(fn, layers, caches, Hkv, hd, page, [&](const Layers& L, bool first) {
    hipLaunchKernelGGL(fork_finish_kernel, dim3(grid_of(4, R * pieces_on_host(Hkv, page, hd) * L.n, R)), dim3(256), 0, stream, a, L, ranges, first);
  });
}

extern "C" int uwc_kv_compact(int layers, void* const* caches, int64_t pages, int page, int Hkv, int hd, const int32_t* table,
                              int64_t table_stride, int width, int B, const int32_t* refs, int32_t* new_table, int32_t* new_refs,
                              void* scratch, uint64_t scratch_bytes, hipStream_t stream) {
  const char* fn = "uwc_kv_compact";
  if (int st = check(fn, layers, caches, pages, page, Hkv, hd, table, table_stride, width, B, refs, scratch, scratch_bytes, 0)) return st;
  if ((B && width && !new_table) || !new_refs) return uwc_fail("%s: null arguments", fn);
  CompactArgs a{table, (long)table_stride, width, B, refs, (int)pages, new_table, new_refs, cut(scratch, pages, 0)};
  const int ranges = (int)ranges_of(pages);
  hipLaunchKernelGGL(compact_plan_kernel, dim3(ranges), dim3(256), 0, stream, a);
  if (int st = uwc_launch_status(fn)) return st;
  return by_layers(fn, layers, caches, Hkv, hd, page, [&](const Layers& L, bool first) {
    // at most half of the pages move
    const long jobs = pages / 2 * pieces_on_host(Hkv, page, hd) * L.n, rows = (pages + (long)B * width + 255) / 256;
    hipLaunchKernelGGL(compact_finish_kernel, dim3(grid_of(8, jobs, rows)), dim3(256), 0, stream, a, L, ranges, first);
  });
}
