// Rows of a table by their numbers, and the gradient of the table:
//
//   y[i] = scale w[ids[i]],   gw[r] = scale sum of gy[i] over the i with ids[i] = r
//
// Both are bound by memory: forward reads the rows that are met and writes y, backward reads gy and writes all of gw.
//
// Numbers repeat, in a point cloud's species hundreds of times, so gw's sums are made by number: the numbers are sorted (stably, with their places), and
// teams of lanes add up the rows of gy of a stretch of them in registers.  Every sum has its order, nothing is added by atomics, and a call repeats bit for
// bit.  The sort has nothing to do with the rows and keeps eight SMs busy; the lookup is launched beside it, and its result is kept for the
// gradient.  The lookup's blocks stay on their SMs until the sort has ended, and where there are more of them than the SMs hold at a time, the rest begin then:
// 32768 rows of 2048 bfloat16 are 8192 blocks, a tenth of which runs beside the sort (a call alone 45 us without the sort, 64 with it).
//
// 32768 rows of 2048 bfloat16 over 65536 entries: sort 23 us, lookup 38, sums 74 (402 MB, 5.4 TB/s), joins 8; a pass with its gradient 148 us for 643 MB,
// 4.3 TB/s, the copy rate being 6.5: rows of 4 KB come from all over memory, and reads and writes take turns.  65536 rows of 112 float32 over 100 entries:
// 9, 19, 14, 20, of a pass of 61, where autograd's hand-over takes 50.
// Steps: a warp per entry that looks through all numbers 15.5 ms and 7.9 ms for these two; sorted numbers 174 and 76; teams of lanes, any alignment and a
// list of what is cut 165 and 64; a sort in one cluster that writes in runs 151 and 60; launched beside the lookup 148.
#include <algorithm>
#include <atomic>
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
__device__ __forceinline__ void look_up(const EmbeddingCall& c, long long i0, int col) {
  using R = typename Raw<V * sizeof(T)>::type;
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

template <class T, int V>
__global__ void __launch_bounds__(kThreads) embedding_kernel(const EmbeddingCall c, Teams t) {
  const long long team = ((long long)blockIdx.x * kThreads + threadIdx.x) / t.lanes, group = team / t.slabs, i0 = group * kRows;
  const int col = ((int)(team - group * t.slabs) * t.lanes + threadIdx.x % t.lanes) * V;
  if (i0 < c.n && col < c.d) look_up<T, V>(c, i0, col);
  await_previous();   // the sort that this kernel is launched beside: what comes after the two follows this one
}

// ---- the numbers in order -----------------------------------------------------------------------------------------------------
//
// Stable radix passes, least significant digit first.  A block ranks a tile of numbers, a warp 32 of them at a time by the lanes that have the same digit, so
// that equal numbers keep their order whatever the timing; puts them in order in shared memory, and writes runs of equal digits: written as they
// come, 65536 numbers on eight SMs took 22 us a pass, a line of the cache for every number.  Where a block's runs go follows from what all blocks have of each
// digit.  Up to 65536 numbers are sorted by the blocks of one cluster, all passes in one launch, which tell each other through shared memory; for more there
// is a launch that counts before each that places.

constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32;
constexpr int kEach = 8;                              // numbers of a thread
constexpr int kTile = kSortThreads * kEach;           // of a block at a time
constexpr int kMaxBits = 10;                          // of a digit, a thread each
constexpr int kClusterMost = 8;
constexpr int kClusterNumbers = kClusterMost * kTile; // that a cluster sorts
constexpr int kSortBlocks = 148;                      // at most, otherwise
static_assert(1 << kMaxBits == kSortThreads, "a thread owns a digit");

struct Sort {
  const void* ids;          // of the first pass
  unsigned *keys[2], *places[2];
  int* counts;              // (blocks, digits)
  long long n, padding, per;   // per: numbers of a block
  int index_bytes, v, passes, bits, blocks;
};
__device__ __forceinline__ unsigned* of_pass(unsigned* const (&two)[2], int pass) { return pass & 1 ? two[1] : two[0]; }
// What does not count has the number v, behind all rows.  What other blocks of a cluster have put down the first cache knows nothing of.
__device__ __forceinline__ unsigned key_of(const Sort& s, int pass, long long i) {
  if (pass > 0) return __ldcg(of_pass(s.keys, pass - 1) + i);
  const long long id = index_at(s.ids, i, s.index_bytes);
  return id < 0 || id >= s.v || id == s.padding ? (unsigned)s.v : (unsigned)id;
}

struct SortShared {
  unsigned short rank[kSortWarps][1 << kMaxBits];
  unsigned key[kTile], place[kTile];
  int start[1 << kMaxBits], to[1 << kMaxBits];   // of a digit: its first place in the tile, and how far from there it goes
  int counts[kClusterMost][1 << kMaxBits];       // of every block of a cluster
  int warp_sum[kSortWarps];
};

// The lanes that are live and have this digit.
__device__ __forceinline__ unsigned lanes_with(unsigned digit, bool live, int bits) {
  unsigned same = __ballot_sync(0xffffffffu, live);
#pragma unroll
  for (int b = 0; b < kMaxBits; b++)
    if (b < bits) {
      const unsigned set = __ballot_sync(0xffffffffu, digit >> b & 1);
      same &= digit >> b & 1 ? set : ~set;
    }
  return same;
}

// The sum of the v of lower threads.
__device__ __forceinline__ int sum_of_lower(SortShared& sh, int v) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  int sum = v;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int o = __shfl_up_sync(0xffffffffu, sum, d);
    if (lane >= d) sum += o;
  }
  if (lane == 31) sh.warp_sum[warp] = sum;
  __syncthreads();
  int lower = lane < warp ? sh.warp_sum[lane] : 0;
#pragma unroll
  for (int d = 16; d; d /= 2) lower += __shfl_xor_sync(0xffffffffu, lower, d);
  __syncthreads();
  return lower + sum - v;
}

// Numbers i0 to i1 of a pass, in a thread's registers.
struct Tile {
  unsigned key[kEach], place[kEach], rank[kEach];   // rank: among the warp's with the same digit
};
// Returns how many of the tile have the thread's digit.
__device__ __forceinline__ int rank_tile(const Sort& s, int pass, long long i0, int count, SortShared& sh, Tile& t) {
  const int digits = 1 << s.bits, shift = pass * s.bits, warp = threadIdx.x / 32, lane = threadIdx.x % 32, each = (count + kSortThreads - 1) / kSortThreads;
  for (int d = lane; d < digits / 2; d += 32) reinterpret_cast<unsigned*>(sh.rank[warp])[d] = 0;
  __syncwarp();
#pragma unroll
  for (int r = 0; r < kEach; r++) {
    const int i = (warp * each + r) * 32 + lane;
    t.key[r] = t.place[r] = t.rank[r] = 0;
    if (r < each && i < count) {
      t.key[r] = key_of(s, pass, i0 + i);
      t.place[r] = pass > 0 ? __ldcg(of_pass(s.places, pass - 1) + i0 + i) : (unsigned)(i0 + i);
    }
  }
#pragma unroll
  for (int r = 0; r < kEach; r++)
    if (r < each) {
      const bool live = (warp * each + r) * 32 + lane < count;
      const unsigned digit = t.key[r] >> shift & (digits - 1), same = lanes_with(digit, live, s.bits);
      const int before = live ? sh.rank[warp][digit] : 0;
      t.rank[r] = before + __popc(same & ((1u << lane) - 1));
      __syncwarp();
      if (live && lane == __ffs(same) - 1) sh.rank[warp][digit] = (unsigned short)(before + __popc(same));
      __syncwarp();
    }
  __syncthreads();
  int sum = 0;
  if ((int)threadIdx.x < digits) {   // over the warps: where each one's begin
#pragma unroll
    for (int w0 = 0; w0 < kSortWarps; w0 += 8) {
      int c[8];
#pragma unroll
      for (int w = 0; w < 8; w++) c[w] = sh.rank[w0 + w][threadIdx.x];
#pragma unroll
      for (int w = 0; w < 8; w++) {
        sh.rank[w0 + w][threadIdx.x] = (unsigned short)sum;
        sum += c[w];
      }
    }
  }
  return sum;
}

// The tile to its places; `sum` as above, `base`: where the first of the thread's digit goes.
__device__ __forceinline__ void place_tile(const Sort& s, int pass, int count, int sum, int base, SortShared& sh, const Tile& t) {
  const int digits = 1 << s.bits, shift = pass * s.bits, warp = threadIdx.x / 32, lane = threadIdx.x % 32, each = (count + kSortThreads - 1) / kSortThreads;
  const int start = sum_of_lower(sh, sum);
  sh.start[threadIdx.x] = start, sh.to[threadIdx.x] = base - start;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kEach; r++)
    if (r < each && (warp * each + r) * 32 + lane < count) {
      const unsigned digit = t.key[r] >> shift & (digits - 1);
      const int at = sh.start[digit] + sh.rank[warp][digit] + t.rank[r];
      sh.key[at] = t.key[r], sh.place[at] = t.place[r];
    }
  __syncthreads();
  unsigned *keys = of_pass(s.keys, pass), *places = of_pass(s.places, pass);
  for (int i = threadIdx.x; i < count; i += kSortThreads) {
    const unsigned key = sh.key[i];
    const int to = sh.to[key >> shift & (digits - 1)] + i;
    keys[to] = key, places[to] = sh.place[i];
  }
  __syncthreads();
}

__device__ __forceinline__ uint32_t at_rank(uint32_t local, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(local), "r"(rank));
  return a;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__global__ void __launch_bounds__(kSortThreads) cluster_sort_kernel(const Sort s) {   // the cluster is the grid
  extern __shared__ __align__(16) unsigned char raw[];
  SortShared& sh = *reinterpret_cast<SortShared*>(raw);
  const int blocks = gridDim.x, block = blockIdx.x, digit = threadIdx.x, digits = 1 << s.bits;
  const long long i0 = min(s.n, block * s.per);
  const int count = (int)(min(s.n, i0 + s.per) - i0);
  let_next_begin();
  cluster_sync();   // all blocks are there
  for (int pass = 0; pass < s.passes; pass++) {
    Tile t;
    const int sum = rank_tile(s, pass, i0, count, sh, t);
    if (digit < digits) {
      const uint32_t mine = (uint32_t)__cvta_generic_to_shared(&sh.counts[block][digit]);
      for (int b = 0; b < blocks; b++) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at_rank(mine, b)), "r"(sum) : "memory");
    }
    cluster_sync();
    int before = 0, all = 0;
    if (digit < digits)
      for (int b = 0; b < blocks; b++) {
        const int c = sh.counts[b][digit];
        before += b < block ? c : 0;
        all += c;
      }
    place_tile(s, pass, count, sum, sum_of_lower(sh, all) + before, sh, t);
    __threadfence();
    cluster_sync();
  }
}

__global__ void __launch_bounds__(kSortThreads) count_kernel(const Sort s, int pass) {
  __shared__ int hist[1 << kMaxBits];
  const int digits = 1 << s.bits, shift = pass * s.bits;
  let_next_begin();
  await_previous();
  hist[threadIdx.x] = 0;
  __syncthreads();
  const long long i0 = blockIdx.x * s.per, i1 = min(s.n, i0 + s.per);
  for (long long i = i0 + threadIdx.x; i < i1; i += kSortThreads) atomicAdd(&hist[key_of(s, pass, i) >> shift & (digits - 1)], 1);
  __syncthreads();
  if ((int)threadIdx.x < digits) s.counts[(blockIdx.x << s.bits) + threadIdx.x] = hist[threadIdx.x];
}

__global__ void __launch_bounds__(kSortThreads) place_kernel(const Sort s, int pass) {
  extern __shared__ __align__(16) unsigned char raw[];
  SortShared& sh = *reinterpret_cast<SortShared*>(raw);
  const int digit = threadIdx.x;
  let_next_begin();
  await_previous();
  int before = 0, all = 0;
  if (digit < 1 << s.bits)
#pragma unroll 8
    for (int b = 0; b < s.blocks; b++) {
      const int c = s.counts[(b << s.bits) + digit];
      before += b < (int)blockIdx.x ? c : 0;
      all += c;
    }
  int base = sum_of_lower(sh, all) + before;
  const long long i1 = min(s.n, (blockIdx.x + 1) * s.per);
  for (long long i0 = blockIdx.x * s.per; i0 < i1; i0 += kTile) {
    const int count = (int)min((long long)kTile, i1 - i0);
    Tile t;
    const int sum = rank_tile(s, pass, i0, count, sh, t);
    place_tile(s, pass, count, sum, base, sh, t);
    base += sum;
  }
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
  int* heads;             // of every stretch: whether something begins there that is cut
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
  const auto head = [&](int cut) {
    if (slab == 0 && lane == 0) a.heads[stretch] = cut;
  };
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
  const long long i1 = i0 + count;
  const bool goes_on = i1 < a.n && a.keys[i1] == cur;
  int cut = 0;
  if (goes_on && whole && !skip && cur < (unsigned)a.v) {
    if (!is_long(a, i1, cur)) {   // the rest of it too
      for (int i = count; i0 + i < a.n; i += kBatch) {
        R raw[kBatch];
        ask(i);
        int live = 0;
#pragma unroll
        for (int j = 0; j < kBatch; j++)
          if (live == j && i0 + i + j < a.n && key[j] == cur) raw[j] = *reinterpret_cast<const R*>(gy + (long long)place[j] * a.d), live++;
#pragma unroll
        for (int j = 0; j < kBatch; j++)
          if (j < live) {
            float g[V];
            unpack<T, V>(raw[j], g);
            add_all(s, s, g);
          }
        if (live < kBatch) break;
      }
      put(false);
      head(0);
      return;
    }
    cut = 1;
  }
  put(goes_on);
  head(cut);
}

template <class T, int V>
__global__ void __launch_bounds__(kThreads, V == 8 ? 2 : 3) reduce_kernel(const Reduce a) {   // eight columns in 80 registers spill: 158 in place of 147 us
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

// What was cut is joined, a row and 32 V of its columns by a warp, or, with many parts, by a block whose warps take parts in turn; either way in the order
// of the parts.  Blocks take every so many-th of the stretches, a thousand at a time.
constexpr int kJoinThreads = 1024, kJoinWarps = kJoinThreads / 32;
constexpr int kFewParts = 16;   // that a warp joins

// The stretch in which what begins in `stretch` and is cut ends; the warp looks at 32 places at a time.
__device__ __forceinline__ long long last_stretch(const Reduce& a, long long stretch, int lane) {
  long long low = (stretch + 1) * a.per, high = a.n;   // low is the row's, high is not
  const unsigned cur = a.keys[low];
  while (high - low > 1) {
    const long long step = (high - low + 32) / 33, at = low + (lane + 1) * step;
    const int same = __popc(__ballot_sync(0xffffffffu, at < high && a.keys[min(at, a.n - 1)] == cur));
    high = min(high, low + (same + 1) * step);
    low += same * step;
  }
  return low / a.per;
}

template <int V>
__device__ __forceinline__ void add_parts(const Reduce& a, long long stretch, long long first, long long last, int step, int col, float (&s)[V]) {
#pragma unroll
  for (int k = 0; k < V; k++) s[k] = 0;
  if (col >= a.d) return;
#pragma unroll 8
  for (long long p = first; p <= last; p += step) {
    float g[V];
    load_part<V>(a.part + (p * 2 + (p == stretch)) * a.d + col, g);
    add_all(s, s, g);
  }
}

template <class T, int V>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const Reduce a) {
  __shared__ float of[kJoinWarps / 2][32 * V];
  __shared__ int heads[kJoinThreads], found[kJoinWarps];
  __shared__ long long last[kJoinThreads];   // of those with many parts
  await_previous();
  const int slabs = (a.d + 32 * V - 1) / (32 * V), lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const long long all = a.stretches * slabs;
  const auto put = [&](long long h, float (&s)[V]) {
    const int col = ((int)(h % slabs) * 32 + lane) * V;
    if (col >= a.d) return;
    mul_all(s, s, a.scale);
    store_vec<T, V>(static_cast<T*>(a.gw) + (long long)a.keys[(h / slabs + 1) * a.per] * a.d + col, s);
  };
  for (long long h0 = blockIdx.x; h0 < all; h0 += (long long)gridDim.x * kJoinThreads) {
    // what is cut among the next thousand of the block's, in order
    const long long mine = h0 + (long long)threadIdx.x * gridDim.x;
    const bool cut = mine < all && a.heads[mine / slabs];
    const unsigned cuts = __ballot_sync(0xffffffffu, cut);
    if (lane == 0) found[warp] = __popc(cuts);
    __syncthreads();
    int before = 0, count = 0;
    for (int w = 0; w < kJoinWarps; w++) before += w < warp ? found[w] : 0, count += found[w];
    if (cut) heads[before + __popc(cuts & ((1u << lane) - 1))] = threadIdx.x;
    __syncthreads();
    for (int k = warp; k < count; k += kJoinWarps) {
      const long long h = h0 + (long long)heads[k] * gridDim.x, stretch = h / slabs, end = last_stretch(a, stretch, lane);
      const bool many = end - stretch >= kFewParts;
      if (lane == 0) last[k] = many ? end : -1;
      if (many) continue;
      float s[V];
      add_parts(a, stretch, stretch, end, 1, ((int)(h % slabs) * 32 + lane) * V, s);
      put(h, s);
    }
    __syncthreads();
    for (int k = 0; k < count; k++) {
      if (last[k] < 0) continue;
      const long long h = h0 + (long long)heads[k] * gridDim.x, stretch = h / slabs;
      float s[V];
      add_parts(a, stretch, stretch + warp, last[k], kJoinWarps, ((int)(h % slabs) * 32 + lane) * V, s);
#pragma unroll
      for (int half = kJoinWarps / 2; half; half /= 2) {
        if (warp >= half && warp < 2 * half)
#pragma unroll
          for (int j = 0; j < V; j++) of[warp - half][j * 32 + lane] = s[j];
        __syncthreads();
        if (warp < half)
#pragma unroll
          for (int j = 0; j < V; j++) s[j] += of[warp][j * 32 + lane];
        __syncthreads();
      }
      if (warp == 0) put(h, s);
    }
    __syncthreads();
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
int launch_forward_as(const EmbeddingCall& c, bool beside, cudaStream_t stream) {
  if (c.d == 0) return GELIB_OK;
  return with_width<T>(c.d, c.ldw, {c.y, c.weight}, [&](auto width) -> int {
    constexpr int V = decltype(width)::value;
    const Teams t = teams_of<V>(c.d);
    const long long blocks = ((c.n + kRows - 1) / kRows * t.slabs * t.lanes + kThreads - 1) / kThreads;
    if (blocks > 0x7fffffffLL) return fail(GELIB_INVALID, "embedding", "too many elements");
    return launch_after("embedding", beside, embedding_kernel<T, V>, dim3((unsigned)blocks), kThreads, 0, stream, c, t);
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

// Blocks of the sort: of a cluster for few numbers, one number a thread at the least; otherwise half a tile.
long long sort_blocks(long long n) {
  if (n <= kClusterNumbers) return std::max(1LL, std::min<long long>(kClusterMost, n / kSortThreads));
  return std::min<long long>(kSortBlocks, 2 * ((n + kTile - 1) / kTile));
}

template <class... P>
int allow_shared(const char* fn, void (*kernel)(P...), std::atomic<uint64_t>* allowed) {   // allowed: devices on which the kernel may have this much shared memory
  int device = 0;
  GELIB_CUDA_TRY(fn, cudaGetDevice(&device));
  const uint64_t bit = device < 64 ? 1ull << device : 0;
  if (allowed->load(std::memory_order_relaxed) & bit) return GELIB_OK;
  GELIB_CUDA_TRY(fn, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(SortShared)));
  allowed->fetch_or(bit, std::memory_order_relaxed);
  return GELIB_OK;
}

int launch_sort(const char* fn, const Sort& s, cudaStream_t stream) {
  static std::atomic<uint64_t> cluster_allowed{0}, place_allowed{0};
  int st;
  if (s.n <= kClusterNumbers) {
    if ((st = allow_shared(fn, cluster_sort_kernel, &cluster_allowed)) != GELIB_OK) return st;
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3(s.blocks), c.blockDim = dim3(kSortThreads), c.dynamicSmemBytes = sizeof(SortShared), c.stream = stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = s.blocks, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
    c.attrs = at, c.numAttrs = 1;
    GELIB_CUDA_TRY(fn, cudaLaunchKernelEx(&c, cluster_sort_kernel, s));
    return launched(fn);
  }
  if ((st = allow_shared(fn, place_kernel, &place_allowed)) != GELIB_OK) return st;
  for (int pass = 0; pass < s.passes; pass++) {
    if ((st = launch_after(fn, pass > 0, count_kernel, dim3(s.blocks), kSortThreads, 0, stream, s, pass)) != GELIB_OK) return st;
    if ((st = launch_after(fn, true, place_kernel, dim3(s.blocks), kSortThreads, sizeof(SortShared), stream, s, pass)) != GELIB_OK) return st;
  }
  return GELIB_OK;
}

// Numbers of a stretch: enough stretches to fill the machine, of whole batches.
template <int V>
int stretch_of(long long n, int d) {
  const Teams t = teams_of<V>(d);
  const long long teams = 148LL * 32 * (32 / t.lanes) / t.slabs;   // of one round
  return (int)std::min(256LL, std::max<long long>(16, (n / std::max(1LL, teams) + kBatch - 1) / kBatch * kBatch));
}

// The state: twice two arrays of numbers, of which the last pass's stay, and the blocks' counts.
Sort sort_of(long long n, int v, void* state, long long* bytes) {
  Sort s = {};
  s.n = n, s.v = v;
  digits_of(v, &s.passes, &s.bits);
  s.blocks = (int)sort_blocks(n);
  s.per = (n + s.blocks - 1) / s.blocks;
  char* at = (char*)state;
  const long long each = up(4 * (n + kBatch));
  for (int i = 0; i < 2; i++) s.keys[i] = (unsigned*)(at + 2 * i * each), s.places[i] = (unsigned*)(at + (2 * i + 1) * each);
  s.counts = (int*)(at + 4 * each);
  if (bytes) *bytes = 4 * each + (n > kClusterNumbers ? up((4LL << s.bits) * s.blocks) : 0);
  return s;
}

long long workspace_of(long long n, int d, int per) {
  const long long stretches = (n + per - 1) / per;
  return up(4 * stretches) + up(stretches * 2 * d * 4);
}

template <class T>
int launch_backward_as(const EmbeddingCall& c, const void* state, char* at, cudaStream_t stream) {
  static const char* fn = "embedding_back";
  return with_width<T>(c.d, c.d, {c.gw, c.gy}, [&](auto width) -> int {
    constexpr int V = decltype(width)::value;
    Reduce a = {};
    a.teams = teams_of<V>(c.d);
    a.per = stretch_of<V>(c.n, c.d);
    const Sort s = sort_of(c.n, c.v, const_cast<void*>(state), nullptr);
    a.keys = s.keys[(s.passes - 1) & 1], a.places = s.places[(s.passes - 1) & 1];
    a.n = c.n, a.stretches = (c.n + a.per - 1) / a.per, a.v = c.v, a.d = c.d, a.scale = c.scale;
    a.heads = (int*)at;
    a.gw = c.gw, a.gy = c.gy, a.part = (float*)(at + up(4 * a.stretches));
    a.blocks = (a.stretches * a.teams.slabs * a.teams.lanes + kThreads - 1) / kThreads;
    const long long blocks = a.blocks + ((long long)c.v + kThreads - 1) / kThreads, cuts = c.n / kShort * ((c.d + 32 * V - 1) / (32 * V));
    if (blocks > 0x7fffffffLL) return fail(GELIB_INVALID, fn, "too many elements");
    int st = launch_after(fn, false, reduce_kernel<T, V>, dim3((unsigned)blocks), kThreads, 0, stream, a);
    if (st != GELIB_OK || c.n <= kShort || a.stretches == 1) return st;   // nothing is cut
    return launch_after(fn, true, join_kernel<T, V>, dim3((unsigned)std::min(cuts, 296LL)), kJoinThreads, 0, stream, a);
  });
}

}  // namespace

long long embedding_state_bytes(long long n, int v) {
  long long bytes;
  sort_of(n, v, nullptr, &bytes);
  return bytes;
}

long long embedding_workspace(long long n, int, int d, int type) {
  long long bytes = 0;
  // the alignment of the call is not known here
  for (int per : {stretch_of<1>(n, d), stretch_of<2>(n, d), stretch_of<4>(n, d), type == GELIB_F32 ? 256 : stretch_of<8>(n, d)})
    bytes = std::max(bytes, workspace_of(n, d, per));
  return bytes;
}

// The sort is made wherever a gradient may be asked for: its numbers are those of this call, which the caller may change before the backward call.
int launch_embedding(const EmbeddingCall& c, void* state, cudaStream_t stream) {
  if (state) {
    Sort s = sort_of(c.n, c.v, state, nullptr);
    s.ids = c.ids, s.padding = c.padding, s.index_bytes = c.index_bytes;
    const int st = launch_sort("embedding", s, stream);
    if (st != GELIB_OK) return st;
  }
  const bool beside = state != nullptr;
  return c.type == GELIB_F32    ? launch_forward_as<float>(c, beside, stream)
         : c.type == GELIB_BF16 ? launch_forward_as<__nv_bfloat16>(c, beside, stream) : launch_forward_as<__half>(c, beside, stream);
}

int launch_embedding_back(const EmbeddingCall& c, const void* state, void* workspace, cudaStream_t stream) {
  char* at = (char*)workspace;
  return c.type == GELIB_F32    ? launch_backward_as<float>(c, state, at, stream)
         : c.type == GELIB_BF16 ? launch_backward_as<__nv_bfloat16>(c, state, at, stream) : launch_backward_as<__half>(c, state, at, stream);
}

}  // namespace gelib_b200
