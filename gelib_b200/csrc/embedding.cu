// Rows of a table by their numbers, and the gradient of the table:
//
//   y[i] = scale w[ids[i]],   gw[r] = scale sum of gy[i] over the i with ids[i] = r
//
// Both are bound by memory: forward reads the rows that are met and writes y, backward reads gy and writes all of gw.
#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <type_traits>

#include "heads.h"

namespace gelib_b200 {

namespace {

constexpr int kThreads = 256;

// Rows are shared out to teams of lanes, side by side over the columns.
struct Teams {
  int lanes, slabs;   // lanes of a team, a power of two up to 32; teams side by side
};
template <int V>
Teams teams_of(int d) {
  Teams t = {1, 0};
  while (t.lanes < 32 && t.lanes * V < d) t.lanes *= 2;
  t.slabs = (d + t.lanes * V - 1) / (t.lanes * V);
  return t;
}

// A team looks up kRows rows that follow one another, so that as many are on their way at a time.
constexpr int kRows = 4;
template <class T, int V>
__global__ void __launch_bounds__(kThreads) embedding_kernel(const EmbeddingCall c, Teams t) {
  using R = typename Raw<V * sizeof(T)>::type;
  const long long team = ((long long)blockIdx.x * kThreads + threadIdx.x) / t.lanes, group = team / t.slabs;
  const int col = ((int)(team - group * t.slabs) * t.lanes + threadIdx.x % t.lanes) * V;
  const long long i0 = group * kRows;
  if (i0 >= c.n || col >= c.d) return;
  long long id[kRows];
  R raw[kRows];
#pragma unroll
  for (int j = 0; j < kRows; j++) id[j] = i0 + j < c.n ? index_at(c.ids, i0 + j, c.index_bytes) : -1;
#pragma unroll
  for (int j = 0; j < kRows; j++)
    if (id[j] >= 0 && id[j] < c.v) raw[j] = *reinterpret_cast<const R*>(static_cast<const T*>(c.weight) + id[j] * c.ldw + col);
#pragma unroll
  for (int j = 0; j < kRows; j++) {
    if (i0 + j >= c.n) break;
    float x[V];
    if (id[j] >= 0 && id[j] < c.v) {
      unpack<T, V>(raw[j], x);
      mul_all(x, x, c.scale);
    } else {
#pragma unroll
      for (int k = 0; k < V; k++) x[k] = NAN;
    }
    store_vec<T, V>(static_cast<T*>(c.y) + (i0 + j) * c.d + col, x);
  }
}

// ---- the numbers in order -----------------------------------------------------------------------------------------------------
//
// Stable radix passes, least significant digit first: a block counts the digits of its stretch of the numbers, the next launch has every block add up what
// others have of each digit, and place its own.  Within a block a warp ranks 32 numbers at a time by the lanes that have the same digit, so
// that equal numbers keep their order whatever the timing.  Few numbers are sorted by one block, all passes in one launch.

constexpr int kSortThreads = 512, kSortWarps = kSortThreads / 32;
constexpr int kEach = 8;                              // numbers of a lane
constexpr int kTile = kSortThreads * kEach;           // of a block at a time
constexpr int kMaxBits = 10;
constexpr int kOneBlock = 2 * kTile;                  // numbers that one block sorts
constexpr int kSortBlocks = 148;                      // at most, otherwise

struct Sort {
  const void* ids;          // of the first pass
  unsigned *keys[2], *places[2];
  int* counts;              // (blocks, digits)
  int* heads;               // its first is set to zero
  long long n, padding, per;   // per: numbers of a block
  int index_bytes, v, passes, bits, blocks;
};
// What does not count has the number v, behind all rows.
__device__ __forceinline__ unsigned key_of(const Sort& s, int pass, long long i) {
  if (pass > 0) return s.keys[(pass - 1) & 1][i];
  const long long id = index_at(s.ids, i, s.index_bytes);
  return id < 0 || id >= s.v || id == s.padding ? (unsigned)s.v : (unsigned)id;
}

struct SortShared {
  unsigned short rank[kSortWarps][1 << kMaxBits];
  int base[1 << kMaxBits];
  int warp_sum[kSortWarps];
};

// sh.base becomes, of every digit, how many numbers have a lower one.
__device__ __forceinline__ void scan_digits(SortShared& sh, int digits) {
  const int t = threadIdx.x, lane = t % 32;
  const int a = 2 * t < digits ? sh.base[2 * t] : 0, b = 2 * t + 1 < digits ? sh.base[2 * t + 1] : 0;
  int sum = a + b;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int o = __shfl_up_sync(0xffffffffu, sum, d);
    if (lane >= d) sum += o;
  }
  if (lane == 31) sh.warp_sum[t / 32] = sum;
  __syncthreads();
  int before = sum - a - b;
  for (int w = 0; w < t / 32; w++) before += sh.warp_sum[w];
  if (2 * t < digits) sh.base[2 * t] = before;
  if (2 * t + 1 < digits) sh.base[2 * t + 1] = before + a;
  __syncthreads();
}

__device__ __forceinline__ void count_digits(const Sort& s, int pass, long long i0, long long i1, int* hist) {
  const int digits = 1 << s.bits, shift = pass * s.bits;
  for (int d = threadIdx.x; d < digits; d += kSortThreads) hist[d] = 0;
  __syncthreads();
  for (long long i = i0 + threadIdx.x; i < i1; i += kSortThreads) atomicAdd(&hist[key_of(s, pass, i) >> shift & (digits - 1)], 1);
  __syncthreads();
}

// Numbers i0 to i1 to their places; sh.base says where the next one of every digit goes.
__device__ __forceinline__ void place_digits(const Sort& s, int pass, long long i0, long long i1, SortShared& sh) {
  const int digits = 1 << s.bits, shift = pass * s.bits, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  unsigned *keys = s.keys[pass & 1], *places = s.places[pass & 1];
  const unsigned* from = s.places[(pass - 1) & 1];
  for (long long t0 = i0; t0 < i1; t0 += kTile) {
    for (int d = threadIdx.x; d < kSortWarps * digits / 2; d += kSortThreads) {
      const int w = d / (digits / 2), at = d % (digits / 2);
      reinterpret_cast<unsigned*>(sh.rank[w])[at] = 0;
    }
    __syncthreads();
    unsigned key[kEach], place[kEach], rank[kEach];
#pragma unroll
    for (int r = 0; r < kEach; r++) {
      const long long i = t0 + (warp * kEach + r) * 32 + lane;
      key[r] = i < i1 ? key_of(s, pass, i) : 0;
      place[r] = i < i1 ? (pass > 0 ? from[i] : (unsigned)i) : 0;
    }
#pragma unroll
    for (int r = 0; r < kEach; r++) {
      const bool live = t0 + (warp * kEach + r) * 32 + lane < i1;
      const unsigned digit = key[r] >> shift & (digits - 1);
      unsigned same = __ballot_sync(0xffffffffu, live);   // the lanes that have this digit
#pragma unroll
      for (int b = 0; b < kMaxBits; b++)
        if (b < s.bits) {
          const unsigned set = __ballot_sync(0xffffffffu, digit >> b & 1);
          same &= digit >> b & 1 ? set : ~set;
        }
      const unsigned short before = live ? sh.rank[warp][digit] : 0;
      rank[r] = before + __popc(same & ((1u << lane) - 1));
      __syncwarp();
      if (live && lane == __ffs(same) - 1) sh.rank[warp][digit] = before + (unsigned short)__popc(same);
      __syncwarp();
    }
    __syncthreads();
    // over the warps: where each one's begin, and how many there are in all
    int total[(1 << kMaxBits) / kSortThreads];
#pragma unroll
    for (int k = 0; k < (1 << kMaxBits) / kSortThreads; k++) {
      const int d = threadIdx.x + k * kSortThreads;
      int sum = 0;
      if (d < digits)
        for (int w = 0; w < kSortWarps; w++) {
          const int c = sh.rank[w][d];
          sh.rank[w][d] = (unsigned short)sum;
          sum += c;
        }
      total[k] = sum;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kEach; r++) {
      if (t0 + (warp * kEach + r) * 32 + lane >= i1) continue;
      const unsigned digit = key[r] >> shift & (digits - 1);
      const int to = sh.base[digit] + sh.rank[warp][digit] + rank[r];
      keys[to] = key[r], places[to] = place[r];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < (1 << kMaxBits) / kSortThreads; k++) {
      const int d = threadIdx.x + k * kSortThreads;
      if (d < digits) sh.base[d] += total[k];
    }
    __syncthreads();
  }
}

__global__ void __launch_bounds__(kSortThreads) sort_kernel(const Sort s) {
  __shared__ SortShared sh;
  let_next_begin();
  if (threadIdx.x == 0) *s.heads = 0;
  for (int pass = 0; pass < s.passes; pass++) {
    count_digits(s, pass, 0, s.n, sh.base);
    scan_digits(sh, 1 << s.bits);
    place_digits(s, pass, 0, s.n, sh);
  }
}

__global__ void __launch_bounds__(kSortThreads) count_kernel(const Sort s, int pass) {
  __shared__ int hist[1 << kMaxBits];
  let_next_begin();
  await_previous();
  if (pass == 0 && blockIdx.x == 0 && threadIdx.x == 0) *s.heads = 0;
  const long long i0 = blockIdx.x * s.per;
  count_digits(s, pass, i0, min(s.n, i0 + s.per), hist);
  for (int d = threadIdx.x; d < 1 << s.bits; d += kSortThreads) s.counts[(blockIdx.x << s.bits) + d] = hist[d];
}

__global__ void __launch_bounds__(kSortThreads) place_kernel(const Sort s, int pass) {
  __shared__ SortShared sh;
  const int digits = 1 << s.bits;
  let_next_begin();
  await_previous();
  int before[(1 << kMaxBits) / kSortThreads];
#pragma unroll
  for (int k = 0; k < (1 << kMaxBits) / kSortThreads; k++) {
    const int d = threadIdx.x + k * kSortThreads;
    int mine = 0, all = 0;
    if (d < digits)
#pragma unroll 8
      for (int b = 0; b < s.blocks; b++) {
        const int c = s.counts[(b << s.bits) + d];
        mine += b < (int)blockIdx.x ? c : 0;
        all += c;
      }
    before[k] = mine;
    if (d < digits) sh.base[d] = all;
  }
  __syncthreads();
  scan_digits(sh, digits);
#pragma unroll
  for (int k = 0; k < (1 << kMaxBits) / kSortThreads; k++) {
    const int d = threadIdx.x + k * kSortThreads;
    if (d < digits) sh.base[d] += before[k];
  }
  __syncthreads();
  const long long i0 = blockIdx.x * s.per;
  place_digits(s, pass, i0, min(s.n, i0 + s.per), sh);
}

// ---- sums of equal numbers ----------------------------------------------------------------------------------------------------
//
// The numbers in order are cut into stretches; a team of lanes, side by side over the columns, adds up the rows of gy of a stretch.  What belongs to one
// row of the table and is not longer than kShort is added by the team in whose stretch it begins; what is longer is cut where stretches are, and
// its parts are joined by another launch in their order.

constexpr int kShort = 32;
constexpr int kBatch = 8;   // rows of gy on their way at a time

struct Reduce {
  const unsigned *keys, *places;
  void* gw;
  const void* gy;
  float* part;            // (stretches, 2, d): of what came before the stretch, of what goes on behind it
  int* heads;             // a count, then the stretches in which something begins that is cut
  long long n, stretches;
  int v, d, per;          // per: numbers of a stretch, a multiple of kBatch
  Teams teams;
  long long blocks;       // that add; the others write zeros to rows that have nothing
  float scale;
};

// V floats of the partial sums, sixteen bytes at a time.
template <int V>
__device__ __forceinline__ void load_part(const float* p, float (&x)[V]) {
  constexpr int W = V < 4 ? V : 4;
#pragma unroll
  for (int k = 0; k < V; k += W) load_vec<float, W>(p + k, reinterpret_cast<float(&)[W]>(x[k]));
}
template <int V>
__device__ __forceinline__ void store_part(float* p, const float (&x)[V]) {
  constexpr int W = V < 4 ? V : 4;
#pragma unroll
  for (int k = 0; k < V; k += W) store_vec<float, W>(p + k, reinterpret_cast<const float(&)[W]>(x[k]));
}

// Whether what has the number at place p, and at the place before, is longer than kShort.
__device__ __forceinline__ bool is_long(const Reduce& a, long long p, unsigned key) {
  if (p >= kShort && a.keys[p - kShort] == key) return true;
  if (p + kShort <= a.n && a.keys[p + kShort - 1] == key) return true;   // p - 1 to p + kShort - 1
  long long b = p - 1;
  while (b > 0 && a.keys[b - 1] == key) b--;
  return b + kShort < a.n && a.keys[b + kShort] == key;
}

template <class T, int V>
__device__ __forceinline__ void add_stretch(const Reduce& a, long long team, int lane) {
  using R = typename Raw<V * sizeof(T)>::type;
  const long long stretch = team / a.teams.slabs, i0 = stretch * a.per;
  const int slab = (int)(team - stretch * a.teams.slabs), col = (slab * a.teams.lanes + lane) * V;
  if (stretch >= a.stretches || col >= a.d) return;
  const T* gy = static_cast<const T*>(a.gy) + col;
  T* gw = static_cast<T*>(a.gw) + col;
  const int count = (int)min((long long)a.per, a.n - i0);
  const unsigned* keys = a.keys + i0;
  unsigned cur = keys[0];
  bool whole = true, skip = false;    // what is being added began here; it is another team's
  if (i0 > 0 && keys[-1] == cur) {
    whole = false;
    skip = !is_long(a, i0, cur);
  }
  float s[V];
#pragma unroll
  for (int k = 0; k < V; k++) s[k] = 0;
  const auto put = [&](bool goes_on) {
    if (cur >= (unsigned)a.v || skip) return;
    if (whole && !goes_on) {
      mul_all(s, s, a.scale);
      store_vec<T, V>(gw + (long long)cur * a.d, s);
    } else {
      store_part<V>(a.part + (stretch * 2 + whole) * a.d + col, s);
    }
  };
  unsigned key[kBatch], place[kBatch];   // of the next rows, asked for a batch ahead
  const auto ask = [&](int i) {
#pragma unroll
    for (int j = 0; j < kBatch; j += 4) {   // there is room for whole batches behind the last number
      const uint4 k4 = *reinterpret_cast<const uint4*>(keys + i + j), p4 = *reinterpret_cast<const uint4*>(a.places + i0 + i + j);
      key[j] = k4.x, key[j + 1] = k4.y, key[j + 2] = k4.z, key[j + 3] = k4.w;
      place[j] = p4.x, place[j + 1] = p4.y, place[j + 2] = p4.z, place[j + 3] = p4.w;
    }
  };
  ask(0);
  for (int i = 0; i < count; i += kBatch) {
    R raw[kBatch];
    unsigned of[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; j++) {
      of[j] = i + j < count ? key[j] : cur;
      if (i + j < count && key[j] < (unsigned)a.v && !(skip && key[j] == cur)) raw[j] = *reinterpret_cast<const R*>(gy + (long long)place[j] * a.d);
    }
    if (i + kBatch < count) ask(i + kBatch);
#pragma unroll
    for (int j = 0; j < kBatch; j++) {
      if (i + j >= count) break;
      if (of[j] != cur) {
        put(false);
        cur = of[j], whole = true, skip = false;
#pragma unroll
        for (int k = 0; k < V; k++) s[k] = 0;
      }
      if (of[j] < (unsigned)a.v && !skip) {
        float g[V];
        unpack<T, V>(raw[j], g);
        add_all(s, s, g);
      }
    }
  }
  if (cur >= (unsigned)a.v || skip) return;
  const long long i1 = i0 + count;
  const bool goes_on = i1 < a.n && a.keys[i1] == cur;
  if (goes_on && whole) {
    if (!is_long(a, i1, cur)) {   // the rest of it too
      for (long long p = i1; p < a.n && a.keys[p] == cur; p++) {
        float g[V];
        load_vec<T, V>(gy + (long long)a.places[p] * a.d, g);
        add_all(s, s, g);
      }
      put(false);
      return;
    }
    if (slab == 0 && lane == 0) a.heads[1 + atomicAdd(a.heads, 1)] = (int)stretch;
  }
  put(goes_on);
}

template <class T, int V>
__global__ void __launch_bounds__(kThreads) reduce_kernel(const Reduce a) {
  let_next_begin();
  await_previous();
  if (blockIdx.x < a.blocks) {
    add_stretch<T, V>(a, ((long long)blockIdx.x * kThreads + threadIdx.x) / a.teams.lanes, threadIdx.x % a.teams.lanes);
    return;
  }
  // zeros: a warp takes 32 rows, of which every lane looks one up
  const int lane = threadIdx.x % 32;
  const long long r0 = ((blockIdx.x - a.blocks) * (kThreads / 32) + threadIdx.x / 32) * 32, r = r0 + lane;
  if (r0 >= a.v) return;
  long long low = 0, high = a.n;   // the first place whose number is r or more
  while (low < high) {
    const long long mid = (low + high) / 2;
    if (a.keys[mid] < (unsigned)r) low = mid + 1;
    else high = mid;
  }
  unsigned none = __ballot_sync(0xffffffffu, r < a.v && (low == a.n || a.keys[low] != (unsigned)r));
  float zero[V];
#pragma unroll
  for (int k = 0; k < V; k++) zero[k] = 0;
  while (none) {
    const long long row = r0 + __ffs(none) - 1;
    none &= none - 1;
    for (int col = lane * V; col < a.d; col += 32 * V) store_vec<T, V>(static_cast<T*>(a.gw) + row * a.d + col, zero);
  }
}

// A block joins the parts of a row and 32 V of its columns, for one after another of what was cut (in whatever order: each is added up by itself): 32
// warps take parts in turn, their sums are added in order.
constexpr int kJoinThreads = 1024, kJoinWarps = kJoinThreads / 32;
template <class T, int V>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const Reduce a) {
  __shared__ float of[kJoinWarps / 2][32 * V];
  await_previous();
  const int slabs = (a.d + 32 * V - 1) / (32 * V), lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const long long all = (long long)*a.heads * slabs;
  for (long long h = blockIdx.x; h < all; h += gridDim.x) {
    const long long stretch = a.heads[1 + h / slabs], i1 = (stretch + 1) * a.per;
    const int col = ((int)(h % slabs) * 32 + lane) * V;
    const unsigned cur = a.keys[i1];
    long long low = i1, high = a.n;   // the first place that is not the row's
    while (low < high) {
      const long long mid = (low + high) / 2;
      if (a.keys[mid] == cur) low = mid + 1;
      else high = mid;
    }
    const long long last = (low - 1) / a.per;
    float s[V];
#pragma unroll
    for (int k = 0; k < V; k++) s[k] = 0;
    if (col < a.d)
#pragma unroll 4
      for (long long p = stretch + warp; p <= last; p += kJoinWarps) {
        float g[V];
        load_part<V>(a.part + (p * 2 + (p == stretch)) * a.d + col, g);
        add_all(s, s, g);
      }
#pragma unroll
    for (int half = kJoinWarps / 2; half; half /= 2) {
      if (warp >= half && warp < 2 * half)
#pragma unroll
        for (int k = 0; k < V; k++) of[warp - half][k * 32 + lane] = s[k];
      __syncthreads();
      if (warp < half)
#pragma unroll
        for (int k = 0; k < V; k++) s[k] += of[warp][k * 32 + lane];
      __syncthreads();
    }
    if (warp == 0 && col < a.d) {
      mul_all(s, s, a.scale);
      store_vec<T, V>(static_cast<T*>(a.gw) + (long long)cur * a.d + col, s);
    }
  }
}

// How many columns go in one access: 16, 8 or 4 bytes of them, or one.  f gets the number as a constant.
template <class T, class F>
int with_width(long long d, long long ld, std::initializer_list<const void*> p, F f) {
  const auto fits = [&](int bytes) {
    bool ok = d * sizeof(T) % bytes == 0 && ld * sizeof(T) % bytes == 0;
    for (const void* q : p) ok = ok && is_aligned(q, bytes);
    return ok;
  };
  if (fits(16)) return f(std::integral_constant<int, 16 / sizeof(T)>());
  if (fits(8)) return f(std::integral_constant<int, 8 / sizeof(T)>());
  if (sizeof(T) == 2 && fits(4)) return f(std::integral_constant<int, sizeof(T) == 2 ? 2 : 1>());
  return f(std::integral_constant<int, 1>());
}

template <class T>
int launch_forward_as(const EmbeddingCall& c, cudaStream_t stream) {
  return with_width<T>(c.d, c.ldw, {c.y, c.weight}, [&](auto width) -> int {
    constexpr int V = decltype(width)::value;
    const Teams t = teams_of<V>(c.d);
    const long long blocks = ((c.n + kRows - 1) / kRows * t.slabs * t.lanes + kThreads - 1) / kThreads;
    if (blocks > 0x7fffffffLL) return fail(GELIB_INVALID, "embedding", "too many elements");
    embedding_kernel<T, V><<<(unsigned)blocks, kThreads, 0, stream>>>(c, t);
    return launched("embedding");
  });
}

long long up(long long bytes) { return (bytes + 255) / 256 * 256; }

// Passes of equal width over the bits of the numbers 0 to v.
void digits_of(int v, int* passes, int* bits) {
  int all = 1;
  while (all < 31 && v >> all) all++;
  *passes = (all + kMaxBits - 1) / kMaxBits;
  *bits = std::max(1, (all + *passes - 1) / *passes);
}

long long sort_blocks(long long n) { return n <= kOneBlock ? 1 : std::min<long long>(kSortBlocks, (n + kTile - 1) / kTile); }

// Numbers of a stretch: enough stretches to fill the machine, of whole batches.
template <int V>
int stretch_of(long long n, int d) {
  const Teams t = teams_of<V>(d);
  const long long teams = 148LL * 32 * (32 / t.lanes) / t.slabs;   // of one round
  return (int)std::min(256LL, std::max<long long>(16, (n / std::max(1LL, teams) + kBatch - 1) / kBatch * kBatch));
}

struct Room {
  long long keys, counts, heads, part, bytes;
};
Room room_of(long long n, int d, int v, int per) {
  int passes, bits;
  digits_of(v, &passes, &bits);
  const long long blocks = sort_blocks(n), stretches = (n + per - 1) / per;
  Room r;
  r.keys = up(4 * (n + kBatch));
  r.counts = blocks > 1 ? up((4LL << bits) * blocks) : 0;
  r.heads = up(4 * (1 + stretches));
  r.part = up(stretches * 2 * d * 4);
  r.bytes = 4 * r.keys + r.counts + r.heads + r.part;
  return r;
}

template <class T>
int launch_backward_as(const EmbeddingCall& c, char* at, cudaStream_t stream) {
  static const char* fn = "embedding_back";
  return with_width<T>(c.d, c.d, {c.gw, c.gy}, [&](auto width) -> int {
    constexpr int V = decltype(width)::value;
    Reduce a = {};
    a.teams = teams_of<V>(c.d);
    a.per = stretch_of<V>(c.n, c.d);
    const Room r = room_of(c.n, c.d, c.v, a.per);
    Sort s = {};
    s.ids = c.ids, s.n = c.n, s.padding = c.padding, s.index_bytes = c.index_bytes, s.v = c.v;
    for (int i = 0; i < 2; i++) s.keys[i] = (unsigned*)(at + 2 * i * r.keys), s.places[i] = (unsigned*)(at + (2 * i + 1) * r.keys);
    s.counts = (int*)(at + 4 * r.keys);
    s.heads = (int*)(at + 4 * r.keys + r.counts);
    digits_of(c.v, &s.passes, &s.bits);
    s.blocks = (int)sort_blocks(c.n);
    s.per = (c.n + s.blocks - 1) / s.blocks;
    int st;
    if (s.blocks == 1) {
      sort_kernel<<<1, kSortThreads, 0, stream>>>(s);
      if ((st = launched(fn)) != GELIB_OK) return st;
    } else {
      for (int pass = 0; pass < s.passes; pass++) {
        if ((st = launch_after(fn, pass > 0, count_kernel, dim3(s.blocks), kSortThreads, 0, stream, s, pass)) != GELIB_OK) return st;
        if ((st = launch_after(fn, true, place_kernel, dim3(s.blocks), kSortThreads, 0, stream, s, pass)) != GELIB_OK) return st;
      }
    }
    a.keys = s.keys[(s.passes - 1) & 1], a.places = s.places[(s.passes - 1) & 1], a.heads = s.heads;
    a.gw = c.gw, a.gy = c.gy, a.part = (float*)(at + 4 * r.keys + r.counts + r.heads);
    a.n = c.n, a.stretches = (c.n + a.per - 1) / a.per, a.v = c.v, a.d = c.d, a.scale = c.scale;
    a.blocks = (a.stretches * a.teams.slabs * a.teams.lanes + kThreads - 1) / kThreads;
    const long long blocks = a.blocks + ((long long)c.v + kThreads - 1) / kThreads, cuts = c.n / kShort * ((c.d + 32 * V - 1) / (32 * V));
    if (blocks > 0x7fffffffLL) return fail(GELIB_INVALID, fn, "too many elements");
    st = launch_after(fn, true, reduce_kernel<T, V>, dim3((unsigned)blocks), kThreads, 0, stream, a);
    if (st != GELIB_OK || c.n <= kShort || a.stretches == 1) return st;   // nothing is cut
    return launch_after(fn, true, join_kernel<T, V>, dim3((unsigned)std::min(cuts, 296LL)), kJoinThreads, 0, stream, a);
  });
}

}  // namespace

long long embedding_workspace(long long n, int v, int d, int type) {
  long long bytes = 0;
  // the alignment of the call is not known here
  for (int per : {stretch_of<1>(n, d), stretch_of<2>(n, d), stretch_of<4>(n, d), type == GELIB_F32 ? 256 : stretch_of<8>(n, d)})
    bytes = std::max(bytes, room_of(n, d, v, per).bytes);
  return bytes;
}

int launch_embedding(const EmbeddingCall& c, cudaStream_t stream) {
  return c.type == GELIB_F32 ? launch_forward_as<float>(c, stream) : c.type == GELIB_BF16 ? launch_forward_as<__nv_bfloat16>(c, stream) : launch_forward_as<__half>(c, stream);
}

int launch_embedding_back(const EmbeddingCall& c, void* workspace, cudaStream_t stream) {
  char* at = (char*)workspace;
  return c.type == GELIB_F32    ? launch_backward_as<float>(c, at, stream)
         : c.type == GELIB_BF16 ? launch_backward_as<__nv_bfloat16>(c, at, stream) : launch_backward_as<__half>(c, at, stream);
}

}  // namespace gelib_b200
