// The product of a dense layer for a handful of rows, one object at a time: what counts is how fast the weights come in.
//
//   y[m][n] = act(sum_k x[m][k] w[k][n] + bias[n]) + residual[m][n],  at most 8 rows
//
// The weights are read once, 16 bytes a lane.  Where a row of the weights holds all n of one k, a lane owns 16 bytes' worth of columns and
// the lanes, warps and blocks of a cluster share k; where it holds all k of one n, a warp owns columns and its lanes share k.  The blocks of a
// cluster add their sums through distributed shared memory in the order of their ranks, so that one launch does it and results repeat.
// 1280 x 1280 bfloat16, one row: 6.3 us a call of the Python function, nearly all of it the call and the launch (3.3 MB of weights take 0.5 us); by the simple product
// with its sums joined by a second launch 37 us.
#include <algorithm>

#include "readout.h"
#include "linear.h"

namespace gelib_b200 {

namespace {

constexpr int kThreads = 256, kWarps = 8;
constexpr int kSms = 148;
constexpr int kKept = 512;   // k of x in shared memory at a time

struct RowsArgs {
  Epilogue e;
  const void *x, *w;
  long long ldx, ldw;
  int M, N, K;
  int per;       // k of a block
};

__device__ __forceinline__ uint32_t rank_of_cluster() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float of_rank(const float* local, uint32_t rank) {
  uint32_t a;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(local)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}

// sums[m * width + c] of every block of the cluster, added up, finished and stored; column c of the block is column n0 + c.
template <class T, int M>
__device__ __forceinline__ void join_and_store(const RowsArgs& a, const float* sums, int width, int n0) {
  const uint32_t ranks = gridDim.y, rank = rank_of_cluster();
  if (ranks > 1) cluster_sync(); else __syncthreads();
  for (int e = threadIdx.x * ranks + rank; e < M * width; e += kThreads * ranks) {
    const int m = e / width, n = n0 + e % width;
    if (m >= a.M || n >= a.N) continue;
    float d[1] = {0};
    for (uint32_t r = 0; r < ranks; r++) d[0] += ranks > 1 ? of_rank(sums + e, r) : sums[e];
    const long long at = (long long)m * a.N + n;
    if (a.e.bias) d[0] += to_float(static_cast<const T*>(a.e.bias)[n]);
    if (a.e.z) static_cast<T*>(a.e.z)[at] = held<T>(d[0]);
    activate(d, a.e.act);
    if (a.e.residual) d[0] += to_float(static_cast<const T*>(a.e.residual)[at]);
    static_cast<T*>(a.e.y)[at] = from_float<T>(d[0]);
  }
  if (ranks > 1) cluster_sync();   // nobody leaves while its sums are read
}

// Rows of w are k's.  A warp has eight lanes side by side and four k's.  X: x's type, T or float.
template <class T, class X, int V, int M>
__global__ void __launch_bounds__(kThreads) rows_by_sum_kernel(RowsArgs a) {
  constexpr int kWidth = 8 * V;
  __shared__ __align__(16) float xs[kKept * M];             // [k][m]
  __shared__ float sums[kWarps * M * kWidth];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, n0 = blockIdx.x * kWidth, n = n0 + lane % 8 * V, mine = warp * 4 + lane / 8;
  const int k0 = blockIdx.y * a.per, k1 = min(a.K, k0 + a.per);
  const X* x = static_cast<const X*>(a.x);
  const T* w = static_cast<const T*>(a.w);
  float s[M][V];
#pragma unroll
  for (int m = 0; m < M; m++)
#pragma unroll
    for (int j = 0; j < V; j++) s[m][j] = 0;
  for (int k = k0; k < k1; k += kKept) {
    const int kept = min(kKept, k1 - k);
    __syncthreads();
    for (int e = threadIdx.x; e < kept * M; e += kThreads) {
      const int q = e % kept, m = e / kept;
      xs[q * M + m] = m < a.M ? to_float(x[m * a.ldx + k + q]) : 0.f;
    }
    __syncthreads();
    if (n < a.N) {
      constexpr int kAhead = 4;
      for (int q = mine; q < kept; q += 32 * kAhead) {
        float v[kAhead][V];
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
          if (q + 32 * i < kept) load_vec<T, V>(w + (long long)(k + q + 32 * i) * a.ldw + n, v[i]);
          else
#pragma unroll
            for (int j = 0; j < V; j++) v[i][j] = 0;
        }
#pragma unroll
        for (int i = 0; i < kAhead; i++)
          if (q + 32 * i < kept) {
#pragma unroll
            for (int m = 0; m < M; m++) {
              const float f = xs[(q + 32 * i) * M + m];
#pragma unroll
              for (int j = 0; j < V; j++) s[m][j] += f * v[i][j];
            }
          }
      }
    }
  }
#pragma unroll
  for (int m = 0; m < M; m++)
#pragma unroll
    for (int j = 0; j < V; j++) {
      s[m][j] += __shfl_xor_sync(0xffffffffu, s[m][j], 8);
      s[m][j] += __shfl_xor_sync(0xffffffffu, s[m][j], 16);
      if (lane < 8) sums[(warp * M + m) * kWidth + lane * V + j] = s[m][j];
    }
  __syncthreads();
  for (int e = threadIdx.x; e < M * kWidth; e += kThreads) {
    float t = 0;
#pragma unroll
    for (int i = 0; i < kWarps; i++) t += sums[i * M * kWidth + e];
    sums[e] = t;       // the first warp's place, which no other thread reads
  }
  join_and_store<T, M>(a, sums, kWidth, n0);
}

// Rows of w are n's.  A warp has C of them; its lanes take V neighbouring k's each.
template <class T, class X, int V, int M, int C>
__global__ void __launch_bounds__(kThreads) rows_across_kernel(RowsArgs a) {
  constexpr int kWidth = kWarps * C;
  __shared__ __align__(16) X xs[M * kKept];                 // [m][k]
  __shared__ float sums[M * kWidth];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, n0 = blockIdx.x * kWidth, n = n0 + warp * C;
  const int k0 = blockIdx.y * a.per, k1 = min(a.K, k0 + a.per);
  const X* x = static_cast<const X*>(a.x);
  const T* w = static_cast<const T*>(a.w);
  float s[C][M];
#pragma unroll
  for (int c = 0; c < C; c++)
#pragma unroll
    for (int m = 0; m < M; m++) s[c][m] = 0;
  for (int k = k0; k < k1; k += kKept) {
    const int kept = min(kKept, k1 - k);
    __syncthreads();
    for (int e = threadIdx.x; e < kept * M; e += kThreads) {
      const int q = e % kept, m = e / kept;
      xs[m * kKept + q] = m < a.M ? x[m * a.ldx + k + q] : from_float<X>(0.f);
    }
    __syncthreads();
    if (n < a.N)
#pragma unroll 2
      for (int q = lane * V; q < kept; q += 32 * V) {
        float v[C][V];
#pragma unroll
        for (int c = 0; c < C; c++) {
          if (n + c < a.N) load_vec<T, V>(w + (n + c) * a.ldw + k + q, v[c]);
          else
#pragma unroll
            for (int j = 0; j < V; j++) v[c][j] = 0;
        }
#pragma unroll
        for (int m = 0; m < M; m++) {
          float f[V];
          constexpr int kOne = V * sizeof(X) > 16 ? 16 / sizeof(X) : V;   // of an access
#pragma unroll
          for (int j = 0; j < V; j += kOne) load_vec<X, kOne>(xs + m * kKept + q + j, reinterpret_cast<float(&)[kOne]>(f[j]));
#pragma unroll
          for (int c = 0; c < C; c++)
#pragma unroll
            for (int j = 0; j < V; j++) s[c][m] += f[j] * v[c][j];
        }
      }
  }
#pragma unroll
  for (int c = 0; c < C; c++)
#pragma unroll
    for (int m = 0; m < M; m++) {
      float t = s[c][m];
#pragma unroll
      for (int d = 16; d; d >>= 1) t += __shfl_xor_sync(0xffffffffu, t, d);
      if (lane == 0) sums[m * kWidth + warp * C + c] = t;
    }
  join_and_store<T, M>(a, sums, kWidth, n0);
}

template <class K>
int launch_rows_as(K kernel, RowsArgs a, int width, int step, cudaStream_t stream) {
  static const char* fn = "linear";
  const int across = (a.N + width - 1) / width;
  // blocks for every SM, of at least one step each
  const int splits = std::max(1, std::min({8, (kSms + across - 1) / across, (a.K + step - 1) / step}));
  a.per = ((a.K + splits - 1) / splits + step - 1) / step * step;
  cudaLaunchConfig_t c = {};
  c.gridDim = dim3(across, (a.K + a.per - 1) / a.per);
  c.blockDim = dim3(kThreads);
  c.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = 1, at[0].val.clusterDim.y = c.gridDim.y, at[0].val.clusterDim.z = 1;
  c.attrs = at;
  c.numAttrs = c.gridDim.y > 1 ? 1 : 0;
  GELIB_CUDA_TRY(fn, cudaLaunchKernelEx(&c, kernel, a));
  return launched(fn);
}

template <class T, class X, int V, int M>
int launch_rows_of(const RowsArgs& a, bool by_sum, cudaStream_t stream) {
  constexpr int C = M >= 4 ? 4 : 1;
  if (by_sum) return launch_rows_as(rows_by_sum_kernel<T, X, V, M>, a, 8 * V, 32, stream);
  return launch_rows_as(rows_across_kernel<T, X, V, M, C>, a, kWarps * C, 32 * V, stream);
}

template <class T, class X, int V>
int launch_rows_wide(const RowsArgs& a, bool by_sum, cudaStream_t stream) {
  if (a.M == 1) return launch_rows_of<T, X, V, 1>(a, by_sum, stream);
  if (a.M <= 4) return launch_rows_of<T, X, V, 4>(a, by_sum, stream);
  return launch_rows_of<T, X, V, 8>(a, by_sum, stream);
}

template <class T, class X>
int launch_rows_type(const RowsArgs& a, const Operand& w, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  const bool wide = is_aligned(a.w, 16) && a.ldw % V == 0 && (w.by_sum ? a.N : a.K) % V == 0;
  return wide ? launch_rows_wide<T, X, V>(a, w.by_sum, stream) : launch_rows_wide<T, X, 1>(a, w.by_sum, stream);
}

}  // namespace

bool takes_rows(const Gemm& g) { return g.M <= 8 && !g.a.by_sum && g.K > 0 && g.K <= 0x7fffffffLL / 2 && (g.N + 7) / 8 <= 0x7fffffffLL; }

int launch_rows(const Gemm& g, cudaStream_t stream) {
  const RowsArgs a = {g.e, g.a.s.base, g.b.s.base, g.a.s.ld, g.b.s.ld, (int)g.M, (int)g.N, (int)g.K, 0};
  if (g.type == GELIB_F32) return launch_rows_type<float, float>(a, g.b, stream);
  if (g.type == GELIB_BF16)
    return g.a.s.in_float ? launch_rows_type<__nv_bfloat16, float>(a, g.b, stream) : launch_rows_type<__nv_bfloat16, __nv_bfloat16>(a, g.b, stream);
  return g.a.s.in_float ? launch_rows_type<__half, float>(a, g.b, stream) : launch_rows_type<__half, __half>(a, g.b, stream);
}

}  // namespace gelib_b200
