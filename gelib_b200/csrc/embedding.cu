// Rows of a table by their numbers, and the gradient of the table:
//
//   y[i] = scale w[ids[i]],   gw[r] = scale sum of gy[i] over the i with ids[i] = r
//
// Both are bound by memory: forward reads the rows that are met and writes y, backward reads gy and writes all of gw.
#include <algorithm>
#include <cmath>

#include "heads.h"

namespace gelib_b200 {

namespace {

constexpr int kThreads = 256;

template <class T, int V>
__global__ void __launch_bounds__(kThreads) embedding_kernel(const EmbeddingCall c) {
  const int chunks = c.d / V;
  const long long all = c.n * chunks;
  for (long long e = (long long)blockIdx.x * kThreads + threadIdx.x; e < all; e += (long long)gridDim.x * kThreads) {
    const long long i = e / chunks, col = (e - i * chunks) * V, id = index_at(c.ids, i, c.index_bytes);
    float x[V];
    if (id >= 0 && id < c.v) {
      load_vec<T, V>(static_cast<const T*>(c.weight) + id * c.ldw + col, x);
      mul_all(x, x, c.scale);
    } else {
#pragma unroll
      for (int k = 0; k < V; k++) x[k] = NAN;
    }
    store_vec<T, V>(static_cast<T*>(c.y) + i * c.d + col, x);
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
      const unsigned same = __match_any_sync(0xffffffffu, live ? digit : 0xffffffffu);
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
  long long n, stretches;
  int v, d, per;          // per: numbers of a stretch, a multiple of kBatch
  int lanes, slabs;       // of a team; teams side by side over the columns
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

// Whether what has the number at place p is longer than kShort, and where it begins as far as kShort places back.
__device__ __forceinline__ bool is_long(const Reduce& a, long long p, unsigned key, long long* begin) {
  long long b = p;
  while (b > 0 && p - b <= kShort && a.keys[b - 1] == key) b--;
  *begin = b;
  return b + kShort < a.n && a.keys[b + kShort] == key;
}

template <class T, int V>
__device__ __forceinline__ void add_stretch(const Reduce& a, long long team, int lane) {
  const long long stretch = team / a.slabs, i0 = stretch * a.per;
  const int col = ((int)(team % a.slabs) * a.lanes + lane) * V;
  if (stretch >= a.stretches || col >= a.d) return;
  const T* gy = static_cast<const T*>(a.gy) + col;
  T* gw = static_cast<T*>(a.gw) + col;
  const long long i1 = min(a.n, i0 + a.per);
  long long i = i0;
  unsigned cur = a.keys[i];
  bool whole = true;    // what is being added began here
  if (i > 0 && a.keys[i - 1] == cur) {
    long long begin;
    if (is_long(a, i, cur, &begin)) whole = false;
    else {
      // another team's
      while (i < i1 && a.keys[i] == cur) i++;
      if (i == i1) return;
      cur = a.keys[i];
    }
  }
  float s[V];
#pragma unroll
  for (int k = 0; k < V; k++) s[k] = 0;
  const auto put = [&](bool goes_on) {
    if (cur >= (unsigned)a.v) return;
    if (whole && !goes_on) {
      mul_all(s, s, a.scale);
      store_vec<T, V>(gw + (long long)cur * a.d, s);
    } else {
      store_part<V>(a.part + (stretch * 2 + whole) * a.d + col, s);
    }
  };
  for (; i < i1; i += kBatch) {
    unsigned key[kBatch];
    typename Raw<V * sizeof(T)>::type raw[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; j++) {
      key[j] = i + j < i1 ? a.keys[i + j] : (unsigned)a.v;
      if (key[j] < (unsigned)a.v) raw[j] = *reinterpret_cast<const typename Raw<V * sizeof(T)>::type*>(gy + (long long)a.places[i + j] * a.d);
    }
#pragma unroll
    for (int j = 0; j < kBatch; j++) {
      if (i + j >= i1) break;
      if (key[j] != cur) {
        put(false);
        cur = key[j], whole = true;
#pragma unroll
        for (int k = 0; k < V; k++) s[k] = 0;
      }
      if (key[j] < (unsigned)a.v) {
        float g[V];
        unpack<T, V>(raw[j], g);
        add_all(s, s, g);
      }
    }
  }
  if (cur >= (unsigned)a.v) return;
  if (i1 == a.n || a.keys[i1] != cur) {
    put(false);
    return;
  }
  if (whole) {
    long long begin = i1;
    while (begin > i0 && a.keys[begin - 1] == cur) begin--;
    if (!(begin + kShort < a.n && a.keys[begin + kShort] == cur)) {   // short: the rest of it too
      for (long long p = i1; p < a.n && a.keys[p] == cur; p++) {
        float g[V];
        load_vec<T, V>(gy + (long long)a.places[p] * a.d, g);
        add_all(s, s, g);
      }
      put(false);
      return;
    }
  }
  put(true);
}

template <class T, int V>
__global__ void __launch_bounds__(kThreads) reduce_kernel(const Reduce a) {
  let_next_begin();
  await_previous();
  if (blockIdx.x < a.blocks) {
    const int teams = kThreads / a.lanes;
    add_stretch<T, V>(a, (long long)blockIdx.x * teams + threadIdx.x / a.lanes, threadIdx.x % a.lanes);
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

// A block joins the parts of one row and 32 V columns, if they begin in its stretch: eight warps take parts in turn, their sums are added in order.
template <class T, int V>
__global__ void __launch_bounds__(kThreads) join_kernel(const Reduce a) {
  __shared__ float of[kThreads / 32][32 * V];
  await_previous();
  const int slabs = (a.d + 32 * V - 1) / (32 * V), lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const long long stretch = blockIdx.x / slabs, i0 = stretch * a.per, i1 = i0 + a.per;
  const int col = ((int)(blockIdx.x % slabs) * 32 + lane) * V;
  if (i1 >= a.n) return;
  const unsigned cur = a.keys[i1];
  if (cur >= (unsigned)a.v || a.keys[i1 - 1] != cur || (a.keys[i0] == cur && i0 > 0 && a.keys[i0 - 1] == cur)) return;   // nothing goes on, or it began before
  long long begin;
  if (!is_long(a, i1, cur, &begin)) return;
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
    for (long long p = stretch + warp; p <= last; p += kThreads / 32) {
      float g[V];
      load_part<V>(a.part + (p * 2 + (p == stretch)) * a.d + col, g);
      add_all(s, s, g);
    }
#pragma unroll
  for (int k = 0; k < V; k++) of[warp][k * 32 + lane] = s[k];
  __syncthreads();
  if (warp > 0 || col >= a.d) return;
#pragma unroll
  for (int w = 1; w < kThreads / 32; w++)
#pragma unroll
    for (int k = 0; k < V; k++) s[k] += of[w][k * 32 + lane];
  mul_all(s, s, a.scale);
  store_vec<T, V>(static_cast<T*>(a.gw) + (long long)cur * a.d + col, s);
}

template <class T>
int launch_forward_as(const EmbeddingCall& c, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  const bool wide = c.d % V == 0 && c.ldw % V == 0 && is_aligned(c.y, 16) && is_aligned(c.weight, 16);
  const long long chunks = c.n * (wide ? c.d / V : c.d);
  const unsigned blocks = (unsigned)std::min((chunks + kThreads - 1) / kThreads, 148LL * 64);
  if (wide) embedding_kernel<T, V><<<blocks, kThreads, 0, stream>>>(c);
  else embedding_kernel<T, 1><<<blocks, kThreads, 0, stream>>>(c);
  return launched("embedding");
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

// Numbers of a stretch: enough stretches to fill the machine a few times over, of whole batches.
int stretch_of(long long n, int d, int V, int* lanes, int* slabs) {
  *lanes = 1;
  while (*lanes < 32 && *lanes * V < d) *lanes *= 2;
  *slabs = (d + *lanes * V - 1) / (*lanes * V);
  const long long teams = 148LL * 32 * (32 / *lanes) / *slabs;   // of one round
  return (int)std::min(256LL, std::max<long long>(16, (n / std::max(1LL, teams) + kBatch - 1) / kBatch * kBatch));
}

struct Room {
  long long keys, counts, part, bytes;
};
Room room_of(long long n, int d, int v, int per) {
  int passes, bits;
  digits_of(v, &passes, &bits);
  const long long blocks = sort_blocks(n);
  Room r;
  r.keys = up(4 * n);
  r.counts = blocks > 1 ? up((4LL << bits) * blocks) : 0;
  r.part = up((n + per - 1) / per * 2 * d * 4);
  r.bytes = 4 * r.keys + r.counts + r.part;
  return r;
}

template <class T>
int launch_backward_as(const EmbeddingCall& c, char* at, cudaStream_t stream) {
  static const char* fn = "embedding_back";
  constexpr int kWide = 16 / sizeof(T);
  const bool wide = c.d % kWide == 0 && is_aligned(c.gw, 16) && is_aligned(c.gy, 16);
  Reduce a = {};
  a.per = stretch_of(c.n, c.d, wide ? kWide : 1, &a.lanes, &a.slabs);
  const Room r = room_of(c.n, c.d, c.v, a.per);
  Sort s = {};
  s.ids = c.ids, s.n = c.n, s.padding = c.padding, s.index_bytes = c.index_bytes, s.v = c.v;
  for (int i = 0; i < 2; i++) s.keys[i] = (unsigned*)(at + 2 * i * r.keys), s.places[i] = (unsigned*)(at + (2 * i + 1) * r.keys);
  s.counts = (int*)(at + 4 * r.keys);
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
  a.keys = s.keys[(s.passes - 1) & 1], a.places = s.places[(s.passes - 1) & 1];
  a.gw = c.gw, a.gy = c.gy, a.part = (float*)(at + 4 * r.keys + r.counts);
  a.n = c.n, a.stretches = (c.n + a.per - 1) / a.per, a.v = c.v, a.d = c.d, a.scale = c.scale;
  const int teams = kThreads / a.lanes;
  a.blocks = (a.stretches * a.slabs + teams - 1) / teams;
  const long long blocks = a.blocks + ((long long)c.v + kThreads - 1) / kThreads, slabs = (c.d + 32 * (wide ? kWide : 1) - 1) / (32 * (wide ? kWide : 1));
  if (blocks > 0x7fffffffLL || a.stretches * slabs > 0x7fffffffLL) return fail(GELIB_INVALID, fn, "too many elements");
  st = launch_after(fn, true, wide ? reduce_kernel<T, kWide> : reduce_kernel<T, 1>, dim3((unsigned)blocks), kThreads, 0, stream, a);
  if (st != GELIB_OK || c.n <= kShort) return st;   // nothing is longer
  return launch_after(fn, true, wide ? join_kernel<T, kWide> : join_kernel<T, 1>, dim3((unsigned)(a.stretches * slabs)), kThreads, 0, stream, a);
}

}  // namespace

long long embedding_workspace(long long n, int v, int d, int type) {
  long long bytes = 0;
  for (int V : {1, 16 / type_bytes(type)}) {   // the alignment of the call is not known here
    int lanes, slabs;
    bytes = std::max(bytes, room_of(n, d, v, stretch_of(n, d, V, &lanes, &slabs)).bytes);
  }
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
