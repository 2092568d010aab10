// A dense layer with its epilogue, and its gradients:
//
//   z = x w + bias,  y = act(z) + residual
//   gz = gy act'(z),  gx = gz w^T,  gw = x^T gz,  gb = sum of gz's rows
//
// Forward is one matrix product whose epilogue adds, activates and rounds once.  Backward is one pass over gy and z for gz and the
// column sums, and two products.  Sums over rows are split over blocks when there are few tiles, as partial sums that are added
// in a fixed order.
#include <algorithm>

#include "linear.h"
#include "readout.h"

namespace gelib_b200 {

namespace {

constexpr int kThreads = 256;
constexpr int kSms = 148;

// ---- simple product: 64 x 64 tiles, 4 x 4 sums per thread, any strides -------------------------------------------------------

constexpr int kTile = 64, kDepth = 16;

template <class T>
__device__ __forceinline__ void finish(const Epilogue& e, long long at, int col, float d) {
  float z[1] = {d};
  if (e.bias) z[0] += to_float(static_cast<const T*>(e.bias)[col]);
  if (e.z) {
    float q = z[0];
    if constexpr (std::is_same_v<T, __half>) q = q < -65504.f ? -65504.f : q > 65504.f ? 65504.f : q;   // an infinity would have no derivative
    static_cast<T*>(e.z)[at] = from_float<T>(q);
  }
  activate(z, e.act);
  if (e.residual) z[0] += to_float(static_cast<const T*>(e.residual)[at]);
  static_cast<T*>(e.y)[at] = from_float<T>(z[0]);
}

// Block (x, y): tile, columns fastest, and part y of the sum.  part: partial sums (parts, M, N), or null.
template <class T>
__global__ void __launch_bounds__(kThreads) simple_gemm_kernel(Gemm g, float* part, long long depth) {
  __shared__ float sa[kDepth][kTile + 4], sb[kDepth][kTile + 4];
  const long long across = (g.N + kTile - 1) / kTile, m0 = blockIdx.x / across * kTile, n0 = blockIdx.x % across * kTile;
  const long long k0 = (long long)blockIdx.y * depth, k1 = min(g.K, k0 + depth);
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  float d[4][4] = {};
  const T *A = static_cast<const T*>(g.a.base), *B = static_cast<const T*>(g.b.base);
  for (long long k = k0; k < k1; k += kDepth) {
    for (int e = threadIdx.x; e < kTile * kDepth; e += kThreads) {
      // the index that is dense in memory runs fastest over the threads
      const int ia = g.a.sk == 1 ? e / kDepth : e % kTile, ka = g.a.sk == 1 ? e % kDepth : e / kTile;
      const int ib = g.b.sk == 1 ? e / kDepth : e % kTile, kb = g.b.sk == 1 ? e % kDepth : e / kTile;
      sa[ka][ia] = m0 + ia < g.M && k + ka < k1 ? to_float(A[(m0 + ia) * g.a.si + (k + ka) * g.a.sk]) : 0.f;
      sb[kb][ib] = n0 + ib < g.N && k + kb < k1 ? to_float(B[(n0 + ib) * g.b.si + (k + kb) * g.b.sk]) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < kDepth; q++) {
      float a[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; i++) a[i] = sa[q][ty * 4 + i], b[i] = sb[q][tx * 4 + i];
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) d[i][j] += a[i] * b[j];
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const long long m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
      if (m >= g.M || n >= g.N) continue;
      if (part) part[((long long)blockIdx.y * g.M + m) * g.N + n] = d[i][j];
      else finish<T>(g.e, m * g.N + n, (int)n, d[i][j]);
    }
}

// The partial sums added up in their order, and the epilogue.
template <class T>
__global__ void __launch_bounds__(kThreads) join_kernel(Epilogue e, const float* part, int parts, long long M, int N) {
  const long long size = M * N;
  for (long long at = (long long)blockIdx.x * kThreads + threadIdx.x; at < size; at += (long long)gridDim.x * kThreads) {
    float d = 0;
    for (int i = 0; i < parts; i++) d += part[i * size + at];
    finish<T>(e, at, (int)(at % N), d);
  }
}

struct Split {
  int parts;
  long long depth;
};
Split split_of(long long M, long long N, long long K) {
  const long long tiles = ((M + kTile - 1) / kTile) * ((N + kTile - 1) / kTile);
  // enough blocks for two on every SM, of at least 256 products deep
  long long parts = std::max(1LL, std::min({kSms * 2 / std::max(1LL, tiles), (K + 255) / 256, 64LL}));
  const long long depth = ((K + parts - 1) / parts + kDepth - 1) / kDepth * kDepth;
  parts = std::max(1LL, depth ? (K + depth - 1) / depth : 1);
  return {(int)parts, depth};
}
long long gemm_workspace(long long M, long long N, long long K) {
  const Split s = split_of(M, N, K);
  return s.parts > 1 ? s.parts * M * N * 4 : 0;
}

template <class T>
int launch_simple(const Gemm& g, float* part, const Split& s, dim3 grid, cudaStream_t stream) {
  simple_gemm_kernel<T><<<grid, kThreads, 0, stream>>>(g, part, s.depth);
  const int st = launched("linear");
  if (st != GELIB_OK || !part) return st;
  join_kernel<T><<<(unsigned)std::min((g.M * g.N + kThreads - 1) / kThreads, 1LL << 20), kThreads, 0, stream>>>(g.e, part, s.parts, g.M, (int)g.N);
  return launched("linear");
}

int launch_gemm(const Gemm& g, void* workspace, cudaStream_t stream) {
  const Split s = split_of(g.M, g.N, g.K);
  float* part = s.parts > 1 ? (float*)workspace : nullptr;
  const long long tiles = ((g.N + kTile - 1) / kTile) * ((g.M + kTile - 1) / kTile);
  if (tiles > 0x7fffffffLL) return fail(GELIB_INVALID, "linear", "too many elements");
  const dim3 grid((unsigned)tiles, s.parts);
  return g.type == GELIB_F32 ? launch_simple<float>(g, part, s, grid, stream)
         : g.type == GELIB_BF16 ? launch_simple<__nv_bfloat16>(g, part, s, grid, stream) : launch_simple<__half>(g, part, s, grid, stream);
}

// ---- gz = gy act'(z) and its column sums ------------------------------------------------------------------------------------------

// Block (x, y): `wide` accesses of V columns, piece y of the rows.  gz may be null (no activation: gy itself), sums too.
template <class T, int V>
__global__ void __launch_bounds__(kThreads) act_back_kernel(T* gz, float* sums, const T* gy, const T* z, long long M, int N, int act, int wide, long long per) {
  __shared__ float chan[kThreads * V];
  const int tx = threadIdx.x % wide, ty = threadIdx.x / wide, high = kThreads / wide;
  const int c = ((int)blockIdx.x * wide + tx) * V;
  const long long r1 = min(M, ((long long)blockIdx.y + 1) * per);
  float s[V];
#pragma unroll
  for (int j = 0; j < V; j++) s[j] = 0;
  if (ty < high && c < N)
    for (long long r = blockIdx.y * per + ty; r < r1; r += high) {
      float g[V];
      load_vec<T, V>(gy + r * N + c, g);
      if (act != GELIB_ACT_NONE) {
        float q[V];
        load_vec<T, V>(z + r * N + c, q);
        activate_back(g, q, act);
        if (gz) store_vec<T, V>(gz + r * N + c, g);
      }
#pragma unroll
      for (int j = 0; j < V; j++) s[j] += g[j];
    }
  if (!sums) return;
#pragma unroll
  for (int j = 0; j < V; j++) chan[threadIdx.x * V + j] = s[j];
  __syncthreads();
  if (ty == 0 && c < N)
#pragma unroll
    for (int j = 0; j < V; j++) {
      float t = 0;
      for (int i = 0; i < high; i++) t += chan[(i * wide + tx) * V + j];
      sums[(long long)blockIdx.y * N + c + j] = t;
    }
}

struct Pieces {
  int V, wide, chunks, parts;
  long long per;
};
Pieces pieces_of(long long M, int N, int type, bool aligned) {
  Pieces p;
  p.V = aligned && N * type_bytes(type) % 16 == 0 ? 16 / type_bytes(type) : 1;
  p.wide = std::min(N / p.V, kThreads);
  p.chunks = (N / p.V + p.wide - 1) / p.wide;
  const int high = kThreads / p.wide;
  const long long parts = std::max(1LL, std::min((M + 4 * high - 1) / (4 * high), (long long)(kSms * 8 + p.chunks - 1) / p.chunks));
  p.per = (M + parts - 1) / parts;
  p.parts = (int)((M + p.per - 1) / p.per);
  return p;
}

template <class T>
int launch_act_back(void* gz, float* sums, const gelib_linear_args& p, const Pieces& q, cudaStream_t stream) {
  constexpr int kWide = 16 / sizeof(T);
  const auto kernel = q.V > 1 ? act_back_kernel<T, kWide> : act_back_kernel<T, 1>;
  kernel<<<dim3(q.chunks, q.parts), kThreads, 0, stream>>>((T*)gz, sums, (const T*)p.gy, (const T*)p.z, p.m, p.n, p.act, q.wide, q.per);
  return launched("linear_back");
}

long long up(long long bytes) { return (bytes + 255) / 256 * 256; }

}  // namespace

long long linear_workspace(const gelib_linear_args& p, bool backward) {
  if (p.m == 0 || p.n == 0) return 0;
  if (!backward) return gemm_workspace(p.m, p.n, p.k);
  long long bytes = 0;
  if (p.act != GELIB_ACT_NONE) bytes += up(p.m * p.n * type_bytes(p.type));
  bytes += up(4LL * p.n * std::max(pieces_of(p.m, p.n, p.type, false).parts, pieces_of(p.m, p.n, p.type, true).parts));
  return bytes + std::max(gemm_workspace(p.m, p.k, p.n), std::max(gemm_workspace(p.k, p.n, p.m), gemm_workspace(p.n, p.k, p.m)));
}

int launch_linear(const gelib_linear_args& p, void* workspace, cudaStream_t stream) {
  Gemm g;
  g.a = {p.x, p.ldx, 1};
  g.b = {p.w, p.w_transposed ? p.ldw : 1, p.w_transposed ? 1 : p.ldw};
  g.e = {p.y, p.z, p.bias, p.residual, p.act};
  g.M = p.m, g.N = p.n, g.K = p.k, g.type = p.type;
  return launch_gemm(g, workspace, stream);
}

int launch_linear_back(const gelib_linear_args& p, void* workspace, cudaStream_t stream) {
  static const char* fn = "linear_back";
  const int width = type_bytes(p.type);
  if (p.m == 0 || p.n == 0) {   // sums of nothing
    if (p.gx && p.m && p.k) GELIB_CUDA_TRY(fn, cudaMemsetAsync(p.gx, 0, (size_t)p.m * p.k * width, stream));
    if (p.gw && p.k && p.n) GELIB_CUDA_TRY(fn, cudaMemsetAsync(p.gw, 0, (size_t)p.k * p.n * width, stream));
    if (p.gb && p.n) GELIB_CUDA_TRY(fn, cudaMemsetAsync(p.gb, 0, (size_t)p.n * width, stream));
    return GELIB_OK;
  }
  char* at = (char*)workspace;
  const void* gz = p.gy;
  const bool act = p.act != GELIB_ACT_NONE;
  if (act) {
    gz = at;
    at += up(p.m * p.n * width);
  }
  float* sums = (float*)at;
  const Pieces q = pieces_of(p.m, p.n, p.type, is_aligned(p.gy, 16) && is_aligned(p.z, 16));
  at += up(4LL * p.n * std::max(pieces_of(p.m, p.n, p.type, false).parts, pieces_of(p.m, p.n, p.type, true).parts));
  if (act || p.gb) {
    void* out = act ? workspace : nullptr;
    float* s = p.gb ? sums : nullptr;
    const int st = p.type == GELIB_F32 ? launch_act_back<float>(out, s, p, q, stream)
                   : p.type == GELIB_BF16 ? launch_act_back<__nv_bfloat16>(out, s, p, q, stream) : launch_act_back<__half>(out, s, p, q, stream);
    if (st != GELIB_OK) return st;
    if (p.gb) {
      const int s2 = launch_sum_parts(p.gb, nullptr, sums, q.parts, p.n, p.type, stream);
      if (s2 != GELIB_OK) return s2;
    }
  }
  Gemm g;
  g.e = {nullptr, nullptr, nullptr, nullptr, GELIB_ACT_NONE};
  g.type = p.type;
  if (p.gx && p.k) {
    g.a = {gz, p.n, 1};
    g.b = {p.w, p.w_transposed ? 1 : p.ldw, p.w_transposed ? p.ldw : 1};
    g.e.y = p.gx;
    g.M = p.m, g.N = p.k, g.K = p.n;
    const int st = launch_gemm(g, at, stream);
    if (st != GELIB_OK) return st;
  }
  if (p.gw && p.k) {
    // in w's own layout: x^T gz, or its transpose gz^T x
    g.a = {p.x, 1, p.ldx};
    g.b = {gz, 1, p.n};
    g.e.y = p.gw;
    g.M = p.k, g.N = p.n, g.K = p.m;
    if (p.w_transposed) {
      std::swap(g.a, g.b);
      std::swap(g.M, g.N);
    }
    return launch_gemm(g, at, stream);
  }
  return GELIB_OK;
}

}  // namespace gelib_b200
