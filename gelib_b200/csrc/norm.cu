// Group norm with an activation, channels last, and its gradients:
//
//   x (b, s, n), channel c of group c / (n / groups); mean and variance over the s positions and the group's channels
//   xh = (x - mean) rstd,  z = xh w + bias,  y = act(z)
//   gz = gy act'(z),  gw = sum gz xh,  gb = sum gz,  gx = rstd (gz w - mean(gz w) - xh mean(gz w xh))
//
// Statistics and sums are float32; the variance is a mean of squares of differences from the mean, not a difference of means, so neither a
// large mean nor an outlier costs digits.  Memory bounds it: a read and a write forward, two reads and a write backward, if the elements that
// share a statistic stay on the SM between its sum and its use.  Three ways of keeping them, by size:
//
//   row    small samples (s = 1 and a group of at most 1024 channels, 512 in float32; or as many numbers in a group, whose row is 1, 2, 4, .. 32
//          accesses): a few lanes of a warp own a (sample, group) in registers
//   tile   a sample's rows of some groups fit a block's shared memory
//   two    larger samples: sums over pieces of a sample, then a second pass over x (and gy) that applies them
//
// Parameter gradients are partial sums per block, added up in a fixed order by a second kernel: results repeat bit for bit.
//
// Measured, forward / backward us (what the bytes take at 6.5 TB/s): rows of 7168 channels in 32 groups, 4096 of them, bfloat16 35 / 54 (18 / 27); no unit is
// full there -- issue slots 56 / 61 %, special functions 52 / 31 % --, the fixed latency of dependent instructions is what 14 warps of an SM wait for.
// 4 x 65536 x 112 float32, in two passes, 70 / 113 (36 / 54 and half as much again for the second reading), memory at 0.75 of its
// rate, a batch of rows on its way at a time; 3000 x 19 x 204 bfloat16, in shared memory, 29 / 56 (7 / 11), the latency of a block's phases.
#include <algorithm>
#include <atomic>

#include "readout.h"
#include "norm.h"

namespace gelib_b200 {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kTileThreads = 128, kTileWarps = kTileThreads / 32;   // of a block that holds a sample: 3000 x 19 x 204 29 us forward, 34 with 256
constexpr int kRowsAhead = 4, kRowsBack = 2;        // of a warp at a time, forward and backward
constexpr int kBlocksAhead = 2, kBlocksBack = 2;    // of an SM
constexpr int kPieceBlocks = 4, kPieceBlocksBack = 2;   // of an SM, where samples are taken in pieces

struct Norm {
  const void *x, *w, *bias, *gy;
  void *y;               // y, or gx
  float *mean, *rstd;    // (b, groups)
  float* part;           // partial sums
  long long b, s;
  int n, groups, cg;     // cg: channels of a group
  float eps;
  int act;
};

__device__ __forceinline__ float lanes_sum(float v, int lanes) {
  for (int d = lanes >> 1; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

// Each of R sums over the lanes, their exchanges side by side.  L: the number of lanes, 0 where it is known at run time only.
template <int L, int R>
__device__ __forceinline__ void lanes_sums(float (&v)[R], int lanes) {
  if constexpr (L > 0) {
#pragma unroll
    for (int d = L >> 1; d; d >>= 1)
#pragma unroll
      for (int r = 0; r < R; r++) v[r] += __shfl_xor_sync(0xffffffffu, v[r], d);
  } else {
    for (int d = lanes >> 1; d; d >>= 1)
#pragma unroll
      for (int r = 0; r < R; r++) v[r] += __shfl_xor_sync(0xffffffffu, v[r], d);
  }
}

template <class T, int V>
__device__ __forceinline__ void load_or(const void* p, long long at, float other, float (&x)[V]) {
  if (p) load_vec<T, V>(static_cast<const T*>(p) + at, x);
  else
#pragma unroll
    for (int k = 0; k < V; k++) x[k] = other;
}

// ---- row: small samples ----------------------------------------------------------------------------------------------------------
// `lanes` lanes (a power of two) own a group: K accesses of V elements each.  A warp keeps its groups, whose weights it holds, and walks samples, R
// at a time: their loads and the exchanges of their sums overlap.  Block (x, y): groups, and every gridDim.y-th set of 8 R samples.
// kMany: samples of several rows, whose group is `vpr` accesses wide, a power of two: a lane has the same channels in all of its rows.
// (4096, 8, 512) in 32 groups, bfloat16: a block per sample took 78 us forward and 131 back.

// Where a lane's k-th access lies from the group's first element, and whether there is one.
struct Spot {
  int row, vec;
};
__device__ __forceinline__ Spot spot_of(bool many, int i, int vpr) { return many ? Spot{i / vpr, i & (vpr - 1)} : Spot{0, i}; }

template <class T, int V>
struct Piece {   // an access as it lies
  typename Raw<V * sizeof(T)>::type raw;
  __device__ __forceinline__ void load(const T* p) { raw = *reinterpret_cast<const typename Raw<V * sizeof(T)>::type*>(p); }
  __device__ __forceinline__ void get(float (&x)[V]) const { unpack<T, V>(raw, x); }
};

template <class T, int V, int K, int R, int L, bool kMany>
__global__ void __launch_bounds__(kThreads, K == 1 ? kBlocksAhead : 1) row_fwd_kernel(Norm a, int lanes, int vpr) {
  if (L > 0) lanes = L;
  const int per = 32 / lanes, lane = threadIdx.x % lanes, warp = threadIdx.x / 32;
  const int g = blockIdx.x * per + (threadIdx.x & 31) / lanes, c0 = g * a.cg;
  const bool live = g < a.groups;
  const long long sample = a.s * a.n;   // its elements
  const float inv = 1.f / ((float)a.s * a.cg);
  constexpr int W = kMany ? 1 : K;
  bool has[K];
  int off[K];
  float w[W][V], bias[W][V];
#pragma unroll
  for (int k = 0; k < K; k++) {
    const Spot at = spot_of(kMany, k * lanes + lane, vpr);
    has[k] = live && at.row < a.s && at.vec * V < a.cg;
    off[k] = at.row * a.n + at.vec * V;
    if (k < W) {
#pragma unroll
      for (int j = 0; j < V; j++) w[k][j] = bias[k][j] = 0;
      if (live && at.vec * V < a.cg) {
        load_or<T, V>(a.w, c0 + at.vec * V, 1.f, w[k]);
        load_or<T, V>(a.bias, c0 + at.vec * V, 0.f, bias[k]);
      }
    }
  }
  const long long step = (long long)gridDim.y * kWarps * R;
  Piece<T, V> next[R][K];
  long long row = ((long long)blockIdx.y * kWarps + warp) * R;
  const T* x = static_cast<const T*>(a.x) + row * sample + c0;
  T* y = static_cast<T*>(a.y) + row * sample + c0;
  auto fetch = [&](long long row) {
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
      for (int k = 0; k < K; k++) {
        if (has[k] && row + r < a.b) next[r][k].load(x + r * sample + off[k]);
        else next[r][k].raw = {};
      }
  };
  if (row < a.b) fetch(row);
  for (; row < a.b; row += step, y += step * sample) {
    float v[R][K][V], mean[R], rstd[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
      mean[r] = 0;
#pragma unroll
      for (int k = 0; k < K; k++) {
        next[r][k].get(v[r][k]);
        mean[r] += sum_of(v[r][k]);
      }
    }
    x += step * sample;
    if (row + step < a.b) fetch(row + step);   // on their way while these rows are worked on
    lanes_sums<L>(mean, lanes);
#pragma unroll
    for (int r = 0; r < R; r++) {
      mean[r] *= inv;
      rstd[r] = 0;
#pragma unroll
      for (int k = 0; k < K; k++) {
        add_all(v[r][k], v[r][k], -mean[r]);
        const float sq = dot_of(v[r][k], v[r][k]);
        if (has[k]) rstd[r] += sq;
      }
    }
    lanes_sums<L>(rstd, lanes);
#pragma unroll
    for (int r = 0; r < R; r++) {
      rstd[r] = rsqrtf(rstd[r] * inv + a.eps);
      if (!live || row + r >= a.b) continue;
      if (a.mean && lane == 0) {
        a.mean[(row + r) * a.groups + g] = mean[r];
        a.rstd[(row + r) * a.groups + g] = rstd[r];
      }
#pragma unroll
      for (int k = 0; k < K; k++)
        if (has[k]) {
          mul_all(v[r][k], v[r][k], rstd[r]);
          fma_all(v[r][k], v[r][k], w[kMany ? 0 : k], bias[kMany ? 0 : k]);
          activate(v[r][k], a.act);
          store_vec<T, V>(y + r * sample + off[k], v[r][k]);
        }
    }
  }
}

// The sums over rows stay in registers; a block's warps have the same groups and add theirs up at the end.
template <class T, int V, int K, int R, int L, bool kMany>
__global__ void __launch_bounds__(kThreads, K == 1 ? kBlocksBack : 1) row_bwd_kernel(Norm a, int lanes, int vpr, int parts) {
  let_next_begin();
  __shared__ float sums[kWarps][2][32 * V];
  if (L > 0) lanes = L;
  const int per = 32 / lanes, lane = threadIdx.x % lanes, warp = threadIdx.x / 32;
  const int g = blockIdx.x * per + (threadIdx.x & 31) / lanes, c0 = g * a.cg;
  const bool live = g < a.groups;
  const long long sample = a.s * a.n;   // its elements
  const float inv = 1.f / ((float)a.s * a.cg);
  constexpr int W = kMany ? 1 : K;
  bool has[K];
  int off[K];
  float w[W][V], bias[W][V], gw[W][V], gb[W][V];
#pragma unroll
  for (int k = 0; k < K; k++) {
    const Spot at = spot_of(kMany, k * lanes + lane, vpr);
    has[k] = live && at.row < a.s && at.vec * V < a.cg;
    off[k] = at.row * a.n + at.vec * V;
    if (k < W) {
#pragma unroll
      for (int j = 0; j < V; j++) w[k][j] = bias[k][j] = gw[k][j] = gb[k][j] = 0;
      if (live && at.vec * V < a.cg) {
        load_or<T, V>(a.w, c0 + at.vec * V, 1.f, w[k]);
        load_or<T, V>(a.bias, c0 + at.vec * V, 0.f, bias[k]);
      }
    }
  }
  const long long step = (long long)gridDim.y * kWarps * R;
  Piece<T, V> px[R][K], pg[R][K];
  float pm[R], pr[R];
  long long row = ((long long)blockIdx.y * kWarps + warp) * R;
  long long at = row * sample + c0, out = at;
  auto fetch = [&](long long row) {
    const T *x = static_cast<const T*>(a.x) + at, *gy = static_cast<const T*>(a.gy) + at;
#pragma unroll
    for (int r = 0; r < R; r++) {
      const bool there = live && row + r < a.b;
      pm[r] = there ? a.mean[(row + r) * a.groups + g] : 0.f;
      pr[r] = there ? a.rstd[(row + r) * a.groups + g] : 0.f;
#pragma unroll
      for (int k = 0; k < K; k++) {
        if (has[k] && row + r < a.b) {
          px[r][k].load(x + r * sample + off[k]);
          pg[r][k].load(gy + r * sample + off[k]);
        } else {
          px[r][k].raw = {};
          pg[r][k].raw = {};
        }
      }
    }
  };
  if (row < a.b) fetch(row);
  for (; row < a.b; row += step, out += step * sample) {
    float h[R][K][V], gz[R][K][V], mean[R], rstd[R], s1[R], s2[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
      mean[r] = pm[r], rstd[r] = pr[r];
#pragma unroll
      for (int k = 0; k < K; k++) px[r][k].get(h[r][k]), pg[r][k].get(gz[r][k]);
    }
    at += step * sample;
    if (row + step < a.b) fetch(row + step);   // on their way while these rows are worked on
#pragma unroll
    for (int r = 0; r < R; r++) {
      s1[r] = s2[r] = 0;
#pragma unroll
      for (int k = 0; k < K; k++) {
        const int q = kMany ? 0 : k;
        float z[V];
        add_all(h[r][k], h[r][k], -mean[r]);   // first the difference: a large mean costs no digits
        mul_all(h[r][k], h[r][k], rstd[r]);
        fma_all(z, h[r][k], w[q], bias[q]);
        activate_back(gz[r][k], z, a.act);     // gy is zero where there is nothing
        add_all(gb[q], gb[q], gz[r][k]);
        fma_all(gw[q], gz[r][k], h[r][k], gw[q]);
        mul_all(gz[r][k], gz[r][k], w[q]);
        s1[r] += sum_of(gz[r][k]);
        s2[r] += dot_of(gz[r][k], h[r][k]);
      }
    }
    if (a.y) {
      lanes_sums<L>(s1, lanes);
      lanes_sums<L>(s2, lanes);
#pragma unroll
      for (int r = 0; r < R; r++) {
        s1[r] *= -inv, s2[r] *= -inv;
#pragma unroll
        for (int k = 0; k < K; k++)
          if (has[k] && row + r < a.b) {
            add_all(gz[r][k], gz[r][k], s1[r]);
            fma_all(gz[r][k], h[r][k], s2[r], gz[r][k]);
            mul_all(gz[r][k], gz[r][k], rstd[r]);
            store_vec<T, V>(static_cast<T*>(a.y) + out + r * sample + off[k], gz[r][k]);
          }
      }
    }
  }
  if (!a.part) return;
  if constexpr (kMany) {   // lanes with the same channels
    for (int d = vpr; d < lanes; d *= 2) {
#pragma unroll
      for (int j = 0; j < V; j++) {
        gw[0][j] += __shfl_xor_sync(0xffffffffu, gw[0][j], d);
        gb[0][j] += __shfl_xor_sync(0xffffffffu, gb[0][j], d);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < W; k++) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < V; j++) {
      sums[warp][0][(threadIdx.x & 31) * V + j] = gw[k][j];
      sums[warp][1][(threadIdx.x & 31) * V + j] = gb[k][j];
    }
    __syncthreads();
    for (int e = threadIdx.x; e < 2 * 32 * V; e += kThreads) {
      const int which = e / (32 * V), q = e % (32 * V), l = q / V;
      const int group = blockIdx.x * per + l / lanes, c = (k * lanes + l % lanes) * V + q % V;
      if (group < a.groups && c < a.cg && (!kMany || l % lanes < vpr)) {
        float t = 0;
#pragma unroll
        for (int i = 0; i < kWarps; i++) t += sums[i][which][q];
        a.part[((long long)which * parts + blockIdx.y) * a.n + group * a.cg + c] = t;
      }
    }
  }
}

// ---- tile: a sample's rows of `gpc` groups in shared memory ----------------------------------------------------------------------
// The channels of the tile are columns of V elements; a thread owns columns and every ty-th row.

struct Columns {
  int cols;      // of the tile, V channels each
  int wide;      // threads side by side: min(cols, kThreads)
  int high;      // rows worked on together
};
__device__ __forceinline__ Columns columns_of(int channels, int V, int threads = kThreads) {
  Columns c;
  c.cols = channels / V;
  c.wide = min(c.cols, threads);
  c.high = threads / c.wide;
  return c;
}

// The groups of a column's V channels: one division, not V.
template <int V>
__device__ __forceinline__ void groups_of(int channel, int cg, int (&g)[V]) {
  int q = channel / cg, rest = channel - q * cg;
#pragma unroll
  for (int j = 0; j < V; j++) {
    g[j] = q;
    if (++rest == cg) rest = 0, q++;
  }
}

// The sum over `high` rows of `channels` of a group's channels, by a warp.
__device__ __forceinline__ float group_sum(const float* chan, int high, int channels, int g, int cg) {
  const int lane = threadIdx.x % 32;
  float t = 0;
  for (int c = lane; c < cg; c += 32)
    for (int i = 0; i < high; i++) t += chan[i * channels + g * cg + c];
  return lanes_sum(t, 32);
}

// The sums of f over a column's rows, one per channel and row of threads, then per group: group[g] = sum.  chan has high * channels floats.
template <int V, class P, class F>
__device__ __forceinline__ void channel_sums(const Columns& c, int rows, int channels, float* chan, P prepare, F f) {
  const int tx = threadIdx.x % c.wide, ty = threadIdx.x / c.wide;
  if (ty < c.high)
    for (int col = tx; col < c.cols; col += c.wide) {
      float sum[V];
#pragma unroll
      for (int j = 0; j < V; j++) sum[j] = 0;
      prepare(col);
      for (int r = ty; r < rows; r += c.high) f(r, col, sum);
#pragma unroll
      for (int j = 0; j < V; j++) chan[ty * channels + col * V + j] = sum[j];
    }
}

__device__ __forceinline__ float warp_total(float v) { return lanes_sum(v, 32); }

template <class T, int V>
__global__ void __launch_bounds__(kTileThreads) tile_fwd_kernel(Norm a, int gpc, int chunks) {
  extern __shared__ __align__(16) unsigned char memory[];
  const int chunk = blockIdx.x % chunks;
  const long long sample = blockIdx.x / chunks;
  const int g0 = chunk * gpc, ng = min(gpc, a.groups - g0), channels = ng * a.cg, c0 = g0 * a.cg, rows = (int)a.s;
  const Columns cl = columns_of(channels, V, kTileThreads);
  T* tile = reinterpret_cast<T*>(memory);
  float* chan = reinterpret_cast<float*>(memory + ((size_t)rows * channels * sizeof(T) + 15) / 16 * 16);
  float* group = chan + max(cl.high * channels, 1);
  const T* x = static_cast<const T*>(a.x) + sample * a.s * a.n + c0;
  const float count = (float)rows * a.cg;
  float mean[V];
  channel_sums<V>(cl, rows, channels, chan, [](int) {}, [&](int r, int col, float (&sum)[V]) {
    using R = typename Raw<V * sizeof(T)>::type;
    const R raw = *reinterpret_cast<const R*>(x + (long long)r * a.n + col * V);
    *reinterpret_cast<R*>(tile + r * channels + col * V) = raw;
    float v[V];
    unpack<T, V>(raw, v);
    add_all(sum, sum, v);
  });
  __syncthreads();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  for (int g = warp; g < ng; g += kTileWarps) {
    const float t = group_sum(chan, cl.high, channels, g, a.cg);
    if (lane == 0) group[g] = t / count;
  }
  __syncthreads();
  auto of_column = [&](int col) {
    int g[V];
    groups_of<V>(col * V, a.cg, g);
#pragma unroll
    for (int j = 0; j < V; j++) mean[j] = group[g[j]];
  };
  channel_sums<V>(cl, rows, channels, chan, of_column, [&](int r, int col, float (&sum)[V]) {
    float v[V];
    load_vec<T, V>(tile + r * channels + col * V, v);
#pragma unroll
    for (int j = 0; j < V; j++) v[j] -= mean[j];
    fma_all(sum, v, v, sum);
  });
  __syncthreads();
  for (int g = warp; g < ng; g += kTileWarps) {
    const float t = group_sum(chan, cl.high, channels, g, a.cg);
    if (lane == 0) {
      const float rstd = rsqrtf(t / count + a.eps);
      group[ng + g] = rstd;
      if (a.mean) {
        a.mean[sample * a.groups + g0 + g] = group[g];
        a.rstd[sample * a.groups + g0 + g] = rstd;
      }
    }
  }
  __syncthreads();
  const int tx = threadIdx.x % cl.wide, ty = threadIdx.x / cl.wide;
  if (ty >= cl.high) return;
  for (int col = tx; col < cl.cols; col += cl.wide) {
    float w[V], bias[V];
    int g[V];
    load_or<T, V>(a.w, c0 + col * V, 1.f, w);
    load_or<T, V>(a.bias, c0 + col * V, 0.f, bias);
    groups_of<V>(col * V, a.cg, g);
#pragma unroll
    for (int j = 0; j < V; j++) {
      mean[j] = group[g[j]];
      w[j] *= group[ng + g[j]];
    }
    for (int r = ty; r < rows; r += cl.high) {
      float v[V];
      load_vec<T, V>(tile + r * channels + col * V, v);
#pragma unroll
      for (int j = 0; j < V; j++) v[j] -= mean[j];
      fma_all(v, v, w, bias);
      activate(v, a.act);
      store_vec<T, V>(static_cast<T*>(a.y) + (sample * a.s + r) * a.n + c0 + col * V, v);
    }
  }
}

// Blocks of one chunk walk the samples; the chunk's parameter sums stay in shared memory.
template <class T, int V>
__global__ void __launch_bounds__(kTileThreads) tile_bwd_kernel(Norm a, int gpc, int parts) {
  let_next_begin();
  extern __shared__ __align__(16) unsigned char memory[];
  const int chunk = blockIdx.x;
  const int g0 = chunk * gpc, ng = min(gpc, a.groups - g0), channels = ng * a.cg, c0 = g0 * a.cg, rows = (int)a.s;
  const Columns cl = columns_of(channels, V, kTileThreads);
  const size_t bytes = ((size_t)rows * channels * sizeof(T) + 15) / 16 * 16;
  T* tx_ = reinterpret_cast<T*>(memory);
  T* tg_ = reinterpret_cast<T*>(memory + bytes);
  float* chan = reinterpret_cast<float*>(memory + 2 * bytes);    // [2][high][channels]
  float* total = chan + 2 * cl.high * channels;                  // [2][channels]
  float* group = total + 2 * channels;                           // [4][ng]: mean, rstd, two means of gradients
  const int tx = threadIdx.x % cl.wide, ty = threadIdx.x / cl.wide, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const float count = (float)rows * a.cg;
  for (int c = threadIdx.x; c < 2 * channels; c += kTileThreads) total[c] = 0;
  for (long long sample = blockIdx.y; sample < a.b; sample += gridDim.y) {
    const long long base = sample * a.s * a.n + c0;
    __syncthreads();
    for (int g = threadIdx.x; g < ng; g += kTileThreads) {
      group[g] = a.mean[sample * a.groups + g0 + g];
      group[ng + g] = a.rstd[sample * a.groups + g0 + g];
    }
    __syncthreads();
    if (ty < cl.high)
      for (int col = tx; col < cl.cols; col += cl.wide) {
        float w[V], bias[V], mean[V], rstd[V], sb[V], sw[V];
        int gr[V];
        load_or<T, V>(a.w, c0 + col * V, 1.f, w);
        load_or<T, V>(a.bias, c0 + col * V, 0.f, bias);
        groups_of<V>(col * V, a.cg, gr);
#pragma unroll
        for (int j = 0; j < V; j++) mean[j] = group[gr[j]], rstd[j] = group[ng + gr[j]], sb[j] = sw[j] = 0;
        for (int r = ty; r < rows; r += cl.high) {
          using R = typename Raw<V * sizeof(T)>::type;
          const int at = r * channels + col * V;
          const long long from = base + (long long)r * a.n + col * V;
          const R rx = *reinterpret_cast<const R*>(static_cast<const T*>(a.x) + from), rg = *reinterpret_cast<const R*>(static_cast<const T*>(a.gy) + from);
          *reinterpret_cast<R*>(tx_ + at) = rx;
          *reinterpret_cast<R*>(tg_ + at) = rg;
          float h[V], g[V], z[V];
          unpack<T, V>(rx, h);
          unpack<T, V>(rg, g);
#pragma unroll
          for (int j = 0; j < V; j++) h[j] -= mean[j];
          mul_all(h, h, rstd);
          fma_all(z, h, w, bias);
          activate_back(g, z, a.act);
          add_all(sb, sb, g);
          fma_all(sw, g, h, sw);
        }
#pragma unroll
        for (int j = 0; j < V; j++) {
          chan[ty * channels + col * V + j] = sw[j];
          chan[(cl.high + ty) * channels + col * V + j] = sb[j];
        }
      }
    __syncthreads();
    for (int c = threadIdx.x; c < channels; c += kTileThreads) {
      float sw = 0, sb = 0;
      for (int i = 0; i < cl.high; i++) sw += chan[i * channels + c], sb += chan[(cl.high + i) * channels + c];
      total[c] += sw;
      total[channels + c] += sb;
      const float w = a.w ? to_float(static_cast<const T*>(a.w)[c0 + c]) : 1.f;
      chan[c] = sw * w;                         // row 0 of its part: read by this thread alone so far
      chan[cl.high * channels + c] = sb * w;
    }
    __syncthreads();
    for (int g = warp; g < ng; g += kTileWarps) {
      float s1 = 0, s2 = 0;
      for (int c = lane; c < a.cg; c += 32) s2 += chan[g * a.cg + c], s1 += chan[cl.high * channels + g * a.cg + c];
      s1 = warp_total(s1), s2 = warp_total(s2);
      if (lane == 0) group[2 * ng + g] = s1 / count, group[3 * ng + g] = s2 / count;
    }
    __syncthreads();
    if (a.y && ty < cl.high)
      for (int col = tx; col < cl.cols; col += cl.wide) {
        float w[V], bias[V], mean[V], rstd[V], s1[V], s2[V];
        int gr[V];
        load_or<T, V>(a.w, c0 + col * V, 1.f, w);
        load_or<T, V>(a.bias, c0 + col * V, 0.f, bias);
        groups_of<V>(col * V, a.cg, gr);
#pragma unroll
        for (int j = 0; j < V; j++) mean[j] = group[gr[j]], rstd[j] = group[ng + gr[j]], s1[j] = group[2 * ng + gr[j]], s2[j] = -group[3 * ng + gr[j]];
        for (int r = ty; r < rows; r += cl.high) {
          float h[V], g[V], z[V];
          load_vec<T, V>(tx_ + r * channels + col * V, h);
          load_vec<T, V>(tg_ + r * channels + col * V, g);
#pragma unroll
          for (int j = 0; j < V; j++) h[j] -= mean[j];
          mul_all(h, h, rstd);
          fma_all(z, h, w, bias);
          activate_back(g, z, a.act);
          mul_all(g, g, w);
#pragma unroll
          for (int j = 0; j < V; j++) g[j] -= s1[j];
          fma_all(g, h, s2, g);
          mul_all(g, g, rstd);
          store_vec<T, V>(static_cast<T*>(a.y) + base + (long long)r * a.n + col * V, g);
        }
      }
  }
  __syncthreads();
  if (a.part)
    for (int c = threadIdx.x; c < 2 * channels; c += kTileThreads)
      a.part[((long long)(c / channels) * parts + blockIdx.y) * a.n + c0 + c % channels] = total[c];
}

// ---- two: pieces of a sample ---------------------------------------------------------------------------------------------------
// A block takes `rows` rows of a sample, all channels.

// Sum, and sum of squares of differences from the piece's own mean, of every group of a piece: part (b, pieces, groups, 2).
template <class T, int V>
__global__ void __launch_bounds__(kThreads, kPieceBlocks) piece_stats_kernel(Norm a, int pieces, int per) {
  let_next_begin();
  extern __shared__ __align__(16) unsigned char memory[];
  const long long sample = blockIdx.x / pieces;
  const int piece = blockIdx.x % pieces;
  const long long r0 = (long long)piece * per;
  const int rows = (int)min((long long)per, a.s - r0);
  const Columns cl = columns_of(a.n, V);
  float* chan = reinterpret_cast<float*>(memory);               // [2][high][n]
  const T* x = static_cast<const T*>(a.x) + (sample * a.s + r0) * a.n;
  const int tx = threadIdx.x % cl.wide, ty = threadIdx.x / cl.wide, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (ty < cl.high)
    for (int col = tx; col < cl.cols; col += cl.wide) {
      // Each batch of rows has its mean first and its squared differences from that after, and joins those before by the difference of the means: no
      // row is a point of reference for the others, so an outlier costs no digits wherever it lies.
      float mean[V], sq[V];
#pragma unroll
      for (int j = 0; j < V; j++) mean[j] = sq[j] = 0;
      const T* at = x + (long long)ty * a.n + col * V;
      const long long step = (long long)cl.high * a.n;
      float count = 0;
      auto batch = [&](auto rows_of) {   // so many rows, on their way together
        constexpr int U = decltype(rows_of)::value;
        Piece<T, V> p[U];
        float m[V], q[V], v[V];
#pragma unroll
        for (int j = 0; j < V; j++) m[j] = q[j] = 0;
#pragma unroll
        for (int u = 0; u < U; u++) p[u].load(at + u * step);
        at += U * step;
#pragma unroll
        for (int u = 0; u < U; u++) {
          p[u].get(v);
          add_all(m, m, v);
        }
        mul_all(m, m, -1.f / U);   // less the mean
#pragma unroll
        for (int u = 0; u < U; u++) {
          p[u].get(v);
          add_all(v, v, m);
          fma_all(q, v, v, q);
        }
        const float share = __fdividef((float)U, count + U);
        add_all(v, mean, m);                 // the means' difference
        fma_all(mean, v, -share, mean);
        mul_all(v, v, v);
        add_all(sq, sq, q);
        fma_all(sq, v, count * share, sq);
        count += U;
      };
      int left = ty < rows ? (rows - ty + cl.high - 1) / cl.high : 0;
      constexpr int kMost = V == 8 ? 4 : 8;   // eight times eight do not fit the registers of four blocks: 2 x 200000 x 512 bfloat16 241 us, 245 with spills
      for (; left >= kMost; left -= kMost) batch(std::integral_constant<int, kMost>{});
      if (left & 4) batch(std::integral_constant<int, 4>{});
      if (left & 2) batch(std::integral_constant<int, 2>{});
      if (left & 1) batch(std::integral_constant<int, 1>{});
#pragma unroll
      for (int j = 0; j < V; j++) {
        chan[ty * a.n + col * V + j] = mean[j];                // of the thread's rows
        chan[(cl.high + ty) * a.n + col * V + j] = sq[j];      // their squared differences from it
      }
    }
  __syncthreads();
  for (int g = warp; g < a.groups; g += kWarps) {
    const int e1 = cl.high * a.cg;
    float t = 0;
    for (int e = lane; e < e1; e += 32) {
      const int i = e / a.cg, mine = i < rows ? (rows - i + cl.high - 1) / cl.high : 0;
      t += mine * chan[i * a.n + g * a.cg + e % a.cg];
    }
    const float mean = warp_total(t) / ((float)rows * a.cg);
    t = 0;
    for (int e = lane; e < e1; e += 32) {
      const int i = e / a.cg, mine = i < rows ? (rows - i + cl.high - 1) / cl.high : 0;
      const float d = chan[i * a.n + g * a.cg + e % a.cg] - mean;
      t += chan[(cl.high + i) * a.n + g * a.cg + e % a.cg] + mine * d * d;
    }
    t = warp_total(t);
    if (lane == 0) {
      float* out = a.part + ((sample * pieces + piece) * a.groups + g) * 2;
      out[0] = mean, out[1] = t;
    }
  }
}

// The pieces' statistics of one (sample, group) as one, by a warp.
__device__ __forceinline__ void join_pieces(const Norm& a, long long sample, int g, int pieces, int per, float* mean_out, float* rstd_out) {
  const int lane = threadIdx.x % 32;
  const float* p = a.part + (sample * pieces * a.groups + g) * 2;
  const long long step = 2LL * a.groups;
  float t = 0;
#pragma unroll 8
  for (int i = lane; i < pieces; i += 32) t += p[i * step] * (float)min((long long)per, a.s - (long long)i * per);
  const float mean = warp_total(t) / (float)a.s;
  t = 0;
  for (int i = lane; i < pieces; i += 32) {
    const float d = p[i * step] - mean;
    t += p[i * step + 1] + d * d * ((float)min((long long)per, a.s - (long long)i * per) * a.cg);
  }
  *mean_out = mean;
  *rstd_out = rsqrtf(warp_total(t) / ((float)a.s * a.cg) + a.eps);
}

template <class T, int V>
__global__ void __launch_bounds__(kThreads, kPieceBlocks) piece_apply_kernel(Norm a, int pieces, int per) {
  await_previous();
  extern __shared__ __align__(16) unsigned char memory[];
  // the pieces that were read last may still be in L2: they are taken first
  const long long block = (long long)gridDim.x - 1 - blockIdx.x;
  const long long sample = block / pieces;
  const int piece = (int)(block % pieces);
  const long long r0 = (long long)piece * per;
  const int rows = (int)min((long long)per, a.s - r0);
  const Columns cl = columns_of(a.n, V);
  float* group = reinterpret_cast<float*>(memory);   // [2][groups]
  const int tx = threadIdx.x % cl.wide, ty = threadIdx.x / cl.wide, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  for (int g = warp; g < a.groups; g += kWarps) {
    float mean, rstd;
    join_pieces(a, sample, g, pieces, per, &mean, &rstd);
    if (lane == 0) {
      group[g] = mean, group[a.groups + g] = rstd;
      if (a.mean && piece == 0) a.mean[sample * a.groups + g] = mean, a.rstd[sample * a.groups + g] = rstd;
    }
  }
  __syncthreads();
  if (ty >= cl.high) return;
  const long long base = (sample * a.s + r0) * a.n;
  for (int col = tx; col < cl.cols; col += cl.wide) {
    float w[V], bias[V], mean[V];
    load_or<T, V>(a.w, col * V, 1.f, w);
    load_or<T, V>(a.bias, col * V, 0.f, bias);
#pragma unroll
    for (int j = 0; j < V; j++) {
      const int g = (col * V + j) / a.cg;
      mean[j] = group[g];
      w[j] *= group[a.groups + g];
    }
    constexpr int U = 4;
    for (int r = ty; r < rows; r += U * cl.high) {
      Piece<T, V> p[U];
#pragma unroll
      for (int u = 0; u < U; u++)
        if (r + u * cl.high < rows) p[u].load(static_cast<const T*>(a.x) + base + (long long)(r + u * cl.high) * a.n + col * V);
#pragma unroll
      for (int u = 0; u < U; u++)
        if (r + u * cl.high < rows) {
          float v[V];
          p[u].get(v);
#pragma unroll
          for (int j = 0; j < V; j++) v[j] = (v[j] - mean[j]) * w[j] + bias[j];
          activate(v, a.act);
          store_vec<T, V>(static_cast<T*>(a.y) + base + (long long)(r + u * cl.high) * a.n + col * V, v);
        }
    }
  }
}

// Rows r, r + high, .. of x and gy as they lie, U of them on their way together: f(x - mean times rstd, gz, z's row).
template <class T, int V, class F>
__device__ __forceinline__ void each_row(const Norm& a, long long base, int rows, int ty, int high, int col, const float (&w)[V], const float (&bias)[V], const float (&mean)[V],
                                         const float (&rstd)[V], F f) {
  constexpr int U = 4;
  const T *x = static_cast<const T*>(a.x) + base + col * V, *gy = static_cast<const T*>(a.gy) + base + col * V;
  for (int r = ty; r < rows; r += U * high) {
    Piece<T, V> px[U], pg[U];
#pragma unroll
    for (int u = 0; u < U; u++)
      if (r + u * high < rows) {
        px[u].load(x + (long long)(r + u * high) * a.n);
        pg[u].load(gy + (long long)(r + u * high) * a.n);
      }
#pragma unroll
    for (int u = 0; u < U; u++)
      if (r + u * high < rows) {
        float h[V], g[V], z[V];
        px[u].get(h);
        pg[u].get(g);
#pragma unroll
        for (int j = 0; j < V; j++) h[j] -= mean[j];
        mul_all(h, h, rstd);
        fma_all(z, h, w, bias);
        activate_back(g, z, a.act);
        f(r + u * high, h, g);
      }
  }
}

// V consecutive floats, V 1 or a multiple of 2.
template <int V>
__device__ __forceinline__ void load_floats(const float* src, float (&x)[V]) {
  constexpr int kOne = V > 4 ? 4 : V;
#pragma unroll
  for (int j = 0; j < V; j += kOne) load_vec<float, kOne>(src + j, reinterpret_cast<float(&)[kOne]>(x[j]));
}
template <int V>
__device__ __forceinline__ void store_floats(float* dst, const float (&x)[V]) {
  constexpr int kOne = V > 4 ? 4 : V;
#pragma unroll
  for (int j = 0; j < V; j += kOne) store_vec<float, kOne>(dst + j, reinterpret_cast<const float(&)[kOne]>(x[j]));
}

// gz xh and gz summed over the rows of a block's pieces, per channel: part (2, blocks, n), or null; and over each piece, times w, per group: back (b, pieces,
// groups, 2).  kWalk: a block takes every gridDim.x-th piece and adds their sums up, else it has one piece.
template <class T, int V, bool kWalk>
__global__ void __launch_bounds__(kThreads, kPieceBlocksBack) piece_back_sums_kernel(Norm a, int pieces, int per, float* back) {
  let_next_begin();
  extern __shared__ __align__(16) unsigned char memory[];
  const Columns cl = columns_of(a.n, V);
  float* chan = reinterpret_cast<float*>(memory);   // [2][high][n]
  const int tx = threadIdx.x % cl.wide, ty = threadIdx.x / cl.wide, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const unsigned items = (unsigned)(a.b * pieces);
  for (unsigned item = blockIdx.x; item < items; item += gridDim.x) {
    const bool first = !kWalk || item == blockIdx.x;
    if (!first) __syncthreads();   // the sums of the piece before have been read
    const long long sample = item / pieces, r0 = (long long)(item % pieces) * per;
    const int rows = (int)min((long long)per, a.s - r0);
    const long long base = (sample * a.s + r0) * a.n;
    if (ty < cl.high)
      for (int col = tx; col < cl.cols; col += cl.wide) {
        float w[V], bias[V], mean[V], rstd[V], sw[V], sb[V];
        load_or<T, V>(a.w, col * V, 1.f, w);
        load_or<T, V>(a.bias, col * V, 0.f, bias);
#pragma unroll
        for (int j = 0; j < V; j++) {
          const long long g = sample * a.groups + (col * V + j) / a.cg;
          mean[j] = a.mean[g], rstd[j] = a.rstd[g], sw[j] = sb[j] = 0;
        }
        each_row<T, V>(a, base, rows, ty, cl.high, col, w, bias, mean, rstd, [&](int, const float (&h)[V], const float (&g)[V]) {
          add_all(sb, sb, g);
          fma_all(sw, g, h, sw);
        });
#pragma unroll
        for (int j = 0; j < V; j++) {
          chan[ty * a.n + col * V + j] = sw[j];
          chan[(cl.high + ty) * a.n + col * V + j] = sb[j];
        }
      }
    __syncthreads();
    for (int e = threadIdx.x; e < 2 * cl.cols; e += kThreads) {
      const int which = e >= cl.cols, q = (e - which * cl.cols) * V;
      float* total = a.part + ((long long)which * gridDim.x + blockIdx.x) * a.n + q;   // this thread's own place, of every piece
      float old[V], t[V];
#pragma unroll
      for (int j = 0; j < V; j++) old[j] = t[j] = 0;
      if (a.part && !first) load_floats(total, old);
      for (int i = 0; i < cl.high; i++) {
        float v[V];
        load_floats(chan + (which * cl.high + i) * a.n + q, v);
        add_all(t, t, v);
      }
      if (a.part) {
        add_all(old, old, t);
        store_floats(total, old);
      }
      if (a.w) {
        float w[V];
        load_vec<T, V>(static_cast<const T*>(a.w) + q, w);
        mul_all(t, t, w);
      }
      store_floats(chan + which * cl.high * a.n + q, t);   // row 0 of its part: read by this thread alone so far
    }
    if (a.y) {
      __syncthreads();
      for (int g = warp; g < a.groups; g += kWarps) {
        float s1 = 0, s2 = 0;
        for (int c = lane; c < a.cg; c += 32) s2 += chan[g * a.cg + c], s1 += chan[cl.high * a.n + g * a.cg + c];
        s1 = warp_total(s1), s2 = warp_total(s2);
        if (lane == 0) {
          float* out = back + ((long long)item * a.groups + g) * 2;
          out[0] = s1, out[1] = s2;
        }
      }
    }
    if (!kWalk) return;
  }
}

template <class T, int V>
__global__ void __launch_bounds__(kThreads, kPieceBlocksBack) piece_back_apply_kernel(Norm a, int pieces, int per, const float* back) {
  let_next_begin();
  await_previous();
  extern __shared__ __align__(16) unsigned char memory[];
  const long long block = (long long)gridDim.x - 1 - blockIdx.x;   // what was read last first
  const long long sample = block / pieces;
  const long long r0 = (block % pieces) * (long long)per;
  const int rows = (int)min((long long)per, a.s - r0);
  const Columns cl = columns_of(a.n, V);
  const int tx = threadIdx.x % cl.wide, ty = threadIdx.x / cl.wide, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const long long base = (sample * a.s + r0) * a.n;
  float* means = reinterpret_cast<float*>(memory);   // [2][groups]
  for (int g = warp; g < a.groups; g += kWarps) {
    float s1 = 0, s2 = 0;
#pragma unroll 8
    for (int i = lane; i < pieces; i += 32) {
      const float2 q = *reinterpret_cast<const float2*>(back + ((sample * pieces + i) * a.groups + g) * 2);
      s1 += q.x, s2 += q.y;
    }
    s1 = warp_total(s1), s2 = warp_total(s2);
    if (lane == 0) means[g] = s1 / ((float)a.s * a.cg), means[a.groups + g] = s2 / ((float)a.s * a.cg);
  }
  __syncthreads();
  if (ty >= cl.high) return;
  for (int col = tx; col < cl.cols; col += cl.wide) {
    float w[V], bias[V], mean[V], rstd[V], s1[V], s2[V];
    load_or<T, V>(a.w, col * V, 1.f, w);
    load_or<T, V>(a.bias, col * V, 0.f, bias);
#pragma unroll
    for (int j = 0; j < V; j++) {
      const int q = (col * V + j) / a.cg;
      const long long g = sample * a.groups + q;
      mean[j] = a.mean[g], rstd[j] = a.rstd[g], s1[j] = means[q], s2[j] = means[a.groups + q];
    }
    each_row<T, V>(a, base, rows, ty, cl.high, col, w, bias, mean, rstd, [&](int r, const float (&h)[V], const float (&g)[V]) {
      float out[V];
#pragma unroll
      for (int j = 0; j < V; j++) out[j] = rstd[j] * (g[j] * w[j] - s1[j] - h[j] * s2[j]);
      store_vec<T, V>(static_cast<T*>(a.y) + base + (long long)r * a.n + col * V, out);
    });
  }
}

// ---- sums over parts -------------------------------------------------------------------------------------------------------------

template <class T>
__global__ void __launch_bounds__(1024) sum_parts_kernel(T* gw, T* gb, const float* sums, int parts, int n) {
  __shared__ float t[32][33];
  await_previous();
  const int c = blockIdx.x * 32 + threadIdx.x;
  T* out = blockIdx.y ? gb : gw;
  if (!out) return;
  const float* p = sums + (long long)blockIdx.y * parts * n;
  float s = 0;
  if (c < n)
#pragma unroll 8
    for (int i = threadIdx.y; i < parts; i += 32) s += p[(long long)i * n + c];
  t[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && c < n) {
    s = 0;
#pragma unroll
    for (int i = 0; i < 32; i++) s += t[i][threadIdx.x];
    out[c] = from_float<T>(s);
  }
}

// ---- which way, and with which sizes ---------------------------------------------------------------------------------------------

constexpr int kSms = 148;
constexpr int kSharedLimit = 200 * 1024;

struct Way {
  enum { kRow, kTile, kTwo } way;
  int V;             // elements of an access
  int lanes, K, R, across, vpr;   // row
  int gpc, chunks;   // tile: groups of a chunk
  size_t shared;     // tile, two
  int parts;         // backward: rows of partial sums
  int pieces, per;   // two
  bool walk;         // two, backward: blocks take several pieces
};

int high_of(int channels, int V, int threads) { return threads / std::min(channels / V, threads); }

Way choose(long long b, long long s, int n, int groups, int type, bool wide16, bool wide8, bool backward) {
  Way w = {};
  const int cg = n / groups, size = type_bytes(type);
  auto fits = [&](int bytes) { return bytes >= size && cg * size % bytes == 0 && (bytes <= size || (bytes == 16 ? wide16 : wide8)); };
  if (s <= 512) {
    const int V = (fits(16) ? 16 : fits(8) ? 8 : size) / size;
    const int across = (cg + V - 1) / V;   // accesses of a row of a group
    const bool even = across <= 32 && (across & (across - 1)) == 0;
    const long long need = across * s;
    if (need <= 128 && (s == 1 || even)) {
      w.way = Way::kRow, w.V = V, w.vpr = across;
      w.lanes = 1;
      while (w.lanes < need && w.lanes < 32) w.lanes *= 2;
      w.K = need <= 32 ? 1 : need <= 64 && s > 1 ? 2 : 4;
      const int across = (groups + 32 / w.lanes - 1) / (32 / w.lanes);
      w.across = across;
      w.R = w.K > 1 ? 1 : backward ? kRowsBack : kRowsAhead;
      // rows for every warp, on as many blocks as the SMs hold
      w.parts = (int)std::max(1LL, std::min((b + kWarps * w.R - 1) / (kWarps * w.R), (long long)(kSms * (backward ? kBlocksBack : kBlocksAhead)) / across));
      return w;
    }
  }
  // an access may hold channels of two groups, but not of two rows or chunks
  auto fits_row = [&](int channels, int bytes) {
    return bytes >= size && n * size % bytes == 0 && channels * size % bytes == 0 && (bytes <= size || (bytes == 16 ? wide16 : wide8));
  };
  auto vector = [&](int channels) { return (fits_row(channels, 16) ? 16 : fits_row(channels, 8) ? 8 : size) / size; };
  auto shared_of = [&](int gpc) {
    const long long channels = (long long)gpc * cg;
    const int V = vector((int)channels), high = high_of((int)channels, V, kTileThreads);
    const long long tile = (s * channels * size + 15) / 16 * 16;
    return backward ? 2 * tile + (2LL * high * channels + 2 * channels + 4 * gpc) * 4 : tile + (high * channels + 2LL * gpc) * 4;
  };
  if (s <= 1 << 20) {
    // whole samples where they leave room for several blocks on an SM and there are enough of them, else fewer groups
    int gpc = groups;
    while (gpc > 1 && (shared_of(gpc) > kSharedLimit / 4 || b * ((groups + gpc - 1) / gpc) < kSms) &&
           (long long)((gpc + 1) / 2) * cg * size >= 64)
      gpc = (gpc + 1) / 2;
    // chunks have to begin on an access's boundary, and the last one may be smaller
    if (shared_of(gpc) <= kSharedLimit) {
      w.way = Way::kTile, w.gpc = gpc, w.chunks = (groups + gpc - 1) / gpc;
      const int last = (groups - (w.chunks - 1) * gpc) * cg;
      w.V = std::min(vector(gpc * cg), vector(last));
      const int high = std::max(high_of(gpc * cg, w.V, kTileThreads), high_of(last, w.V, kTileThreads));
      const long long channels = (long long)gpc * cg, tile = (s * channels * size + 15) / 16 * 16;
      w.shared = backward ? 2 * tile + (2LL * high * channels + 2 * channels + 4 * gpc) * 4 : tile + (high * channels + 2LL * gpc) * 4;
      if (w.shared <= (size_t)kSharedLimit) {
        const long long resident = std::max(1LL, std::min(2048LL / kTileThreads, (long long)(220 * 1024) / (long long)(w.shared + 1024)));
        w.parts = (int)std::max(1LL, std::min(b, (kSms * resident + w.chunks - 1) / w.chunks));
        return w;
      }
    }
  }
  w.way = Way::kTwo, w.V = vector(n);
  const int high = high_of(n, w.V, kThreads);
  w.shared = std::max(2LL * high * n, 2LL * groups) * 4;
  // as many blocks as the SMs hold at a time, so that all of them end together; rows enough in a piece that its sums are few beside it
  const long long wanted = std::max(1LL, kSms * (backward ? kPieceBlocksBack : kPieceBlocks) / b);
  w.per = (int)std::min((long long)1 << 24, std::max({(s + wanted - 1) / wanted, (long long)4 * high, std::min(s, (long long)16)}));
  w.pieces = (int)((s + w.per - 1) / w.per);
  // Partial sums of the parameters' gradients are 8 bytes a channel: a row of them for each piece, or for each of as many blocks as the SMs hold, which then walk
  // the pieces.  They walk where a row would be more than a sixteenth of its piece (4000 x 4 x 7168 bfloat16 backward 452 us, 683 with a row each), and where
  // there are so many pieces that the workspace would grow with the batch.  Else the walk costs more than the rows (500 x 900 x 520 bfloat16
  // 710 us, 686 with a row each).
  const long long samples = b * w.pieces, wave = (long long)kSms * kPieceBlocksBack;
  w.walk = samples > 8 * wave || (samples > wave && std::min(s, (long long)w.per) * size < 128);
  w.parts = (int)std::min(w.walk ? wave : samples, 0x7fffffffLL);
  return w;
}

bool wide_at(std::initializer_list<const void*> p, int bytes) {
  for (const void* q : p)
    if (!is_aligned(q, bytes)) return false;
  return true;
}

template <class T, class F>
int with_vector(int V, F f) {
  if constexpr (sizeof(T) == 4) {
    if (V == 4) return f(std::integral_constant<int, 4>{});
    if (V == 2) return f(std::integral_constant<int, 2>{});
  } else {
    if (V == 8) return f(std::integral_constant<int, 8>{});
    if (V == 4) return f(std::integral_constant<int, 4>{});
  }
  return f(std::integral_constant<int, 1>{});
}

template <class F>
int with_type(int type, F f) {
  if (type == GELIB_F32) return f((float*)nullptr);
  if (type == GELIB_BF16) return f((__nv_bfloat16*)nullptr);
  return f((__half*)nullptr);
}

// More shared memory than a block has by itself.  The limit belongs to the kernel, in every thread of the process: it is set once on a device, to the most
// that any call takes, and never lowered under another thread's launch.
template <auto kernel>
int room(const char* fn, size_t bytes) {
  if (bytes <= 48 * 1024) return GELIB_OK;
  static std::atomic<uint64_t> allowed{0};   // devices on which it is set
  int device = 0;
  GELIB_CUDA_TRY(fn, cudaGetDevice(&device));
  const uint64_t bit = device < 64 ? 1ull << device : 0;
  if (allowed.load(std::memory_order_relaxed) & bit) return GELIB_OK;
  GELIB_CUDA_TRY(fn, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSharedLimit));
  allowed.fetch_or(bit, std::memory_order_relaxed);
  return GELIB_OK;
}

}  // namespace

int launch_sum_parts(void* gw, void* gb, const float* sums, int parts, int n, int type, cudaStream_t stream) {
  if (!gw && !gb) return GELIB_OK;
  return with_type(type, [&](auto* t) -> int {
    using T = std::remove_pointer_t<decltype(t)>;
    return launch_after("sum_parts", true, sum_parts_kernel<T>, dim3((n + 31) / 32, 2), dim3(32, 32), 0, stream, (T*)gw, (T*)gb, sums, parts, n);
  });
}

long long group_norm_workspace(long long b, long long s, int n, int groups, int type, bool backward) {
  // alignment may only make accesses narrower; what depends on them is bounded by the narrowest
  long long most = 0;
  for (int k = 0; k < 3; k++) {
    const Way w = choose(b, s, n, groups, type, k == 2, k >= 1, backward);
    long long floats = 0;
    if (w.way == Way::kTwo) floats = 2LL * b * w.pieces * groups + (backward ? 2LL * w.parts * n : 0);
    else if (backward) floats = 2LL * w.parts * n;
    most = std::max(most, floats);
  }
  return most * 4;
}

int launch_group_norm(const GroupNormCall& c, cudaStream_t stream) {
  const char* fn = c.gy ? "group_norm_back" : "group_norm";
  const bool back = c.gy != nullptr;
  const Way w = choose(c.b, c.s, c.n, c.groups, c.type, wide_at({c.x, c.w, c.bias, c.gy, c.y}, 16), wide_at({c.x, c.w, c.bias, c.gy, c.y}, 8), back);
  Norm a = {c.x, c.w, c.bias, c.gy, c.y, c.mean, c.rstd, c.workspace, c.b, c.s, c.n, c.groups, c.n / c.groups, c.eps, c.act};
  const bool sums = c.gw || c.gb;
  if ((back || w.way != Way::kTwo) && !sums) a.part = nullptr;   // the forward in two passes keeps its statistics there
  const long long samples = w.way == Way::kTwo ? c.b * w.pieces : w.way == Way::kTile ? c.b * w.chunks : 1;
  if (samples > 0x7fffffffLL) return fail(GELIB_INVALID, fn, "too many samples");
  const int st = with_type(c.type, [&](auto* t) -> int {
    using T = std::remove_pointer_t<decltype(t)>;
    return with_vector<T>(w.V, [&](auto v) -> int {
      constexpr int V = decltype(v)::value;
      int st;
      if (w.way == Way::kRow) {
        const dim3 grid(w.across, w.parts);
        const bool many = c.s > 1;
        if (!back) {
          const auto kernel = many ? (w.K == 4   ? row_fwd_kernel<T, V, 4, 1, 32, true>
                                      : w.K == 2 ? row_fwd_kernel<T, V, 2, 1, 32, true>
                                      : w.lanes == 32 ? row_fwd_kernel<T, V, 1, kRowsAhead, 32, true> : row_fwd_kernel<T, V, 1, kRowsAhead, 0, true>)
                                   : (w.K == 4 ? row_fwd_kernel<T, V, 4, 1, 32, false>
                                      : w.lanes == 32 ? row_fwd_kernel<T, V, 1, kRowsAhead, 32, false> : row_fwd_kernel<T, V, 1, kRowsAhead, 0, false>);
          kernel<<<grid, kThreads, 0, stream>>>(a, w.lanes, w.vpr);
        } else {
          const auto kernel = many ? (w.K == 4   ? row_bwd_kernel<T, V, 4, 1, 32, true>
                                      : w.K == 2 ? row_bwd_kernel<T, V, 2, 1, 32, true>
                                      : w.lanes == 32 ? row_bwd_kernel<T, V, 1, kRowsBack, 32, true> : row_bwd_kernel<T, V, 1, kRowsBack, 0, true>)
                                   : (w.K == 4 ? row_bwd_kernel<T, V, 4, 1, 32, false>
                                      : w.lanes == 32 ? row_bwd_kernel<T, V, 1, kRowsBack, 32, false> : row_bwd_kernel<T, V, 1, kRowsBack, 0, false>);
          kernel<<<grid, kThreads, 0, stream>>>(a, w.lanes, w.vpr, w.parts);
        }
        return launched(fn);
      }
      if (w.way == Way::kTile) {
        if (!back) {
          if ((st = room<tile_fwd_kernel<T, V>>(fn, w.shared)) != GELIB_OK) return st;
          tile_fwd_kernel<T, V><<<(unsigned)samples, kTileThreads, w.shared, stream>>>(a, w.gpc, w.chunks);
        } else {
          if ((st = room<tile_bwd_kernel<T, V>>(fn, w.shared)) != GELIB_OK) return st;
          tile_bwd_kernel<T, V><<<dim3(w.chunks, w.parts), kTileThreads, w.shared, stream>>>(a, w.gpc, w.parts);
        }
        return launched(fn);
      }
      if (w.shared > (size_t)kSharedLimit) return fail(GELIB_INVALID, fn, "too many channels");  // not up to GELIB_NORM_MAX_CHANNELS
      if (!back) {
        if ((st = room<piece_stats_kernel<T, V>>(fn, w.shared)) != GELIB_OK) return st;
        piece_stats_kernel<T, V><<<(unsigned)samples, kThreads, w.shared, stream>>>(a, w.pieces, w.per);
        if ((st = launched(fn)) != GELIB_OK) return st;
        const size_t shared = 2ULL * c.groups * 4;
        if ((st = room<piece_apply_kernel<T, V>>(fn, shared)) != GELIB_OK) return st;
        return launch_after(fn, true, piece_apply_kernel<T, V>, dim3((unsigned)samples), kThreads, shared, stream, a, w.pieces, w.per);
      }
      float* back = c.workspace + 2LL * w.parts * c.n;
      if (w.walk) {
        if ((st = room<piece_back_sums_kernel<T, V, true>>(fn, w.shared)) != GELIB_OK) return st;
        piece_back_sums_kernel<T, V, true><<<w.parts, kThreads, w.shared, stream>>>(a, w.pieces, w.per, back);
      } else {
        if ((st = room<piece_back_sums_kernel<T, V, false>>(fn, w.shared)) != GELIB_OK) return st;
        piece_back_sums_kernel<T, V, false><<<w.parts, kThreads, w.shared, stream>>>(a, w.pieces, w.per, back);
      }
      if ((st = launched(fn)) != GELIB_OK || !a.y) return st;
      const size_t shared = 2ULL * c.groups * 4;
      if ((st = room<piece_back_apply_kernel<T, V>>(fn, shared)) != GELIB_OK) return st;
      return launch_after(fn, true, piece_back_apply_kernel<T, V>, dim3((unsigned)samples), kThreads, shared, stream, a, w.pieces, w.per, (const float*)back);
    });
  });
  if (st != GELIB_OK || !back) return st;
  return launch_sum_parts(c.gw, c.gb, c.workspace, w.parts, c.n, c.type, stream);
}

}  // namespace gelib_b200
