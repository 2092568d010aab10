// A dense layer with its epilogue, and its gradients:
//
//   z = x w + bias,  y = act(z) + residual
//   gz = gy act'(z),  gx = gz w^T,  gw = x^T gz,  gb = sum of gz's rows
//
// Forward is one matrix product whose epilogue adds, activates and rounds once.  Backward is one pass over gy and z for gz and the
// column sums, and two products.  Sums over rows are split over blocks when there are few tiles, as partial sums that are added
// in a fixed order.
#include <algorithm>

#include "readout.h"
#include "linear.h"
#include "plan.h"

namespace gelib_b200 {

namespace {

constexpr int kThreads = 256;
constexpr int kSms = 148;

// Element (i, k) of an operand at base[i * si + k * sk], i the row of A or the column of B.
struct Strided {
  const void* base;
  long long si, sk;
};
Strided strided(const Operand& o) { return {o.s.base, o.by_sum ? 1 : o.s.ld, o.by_sum ? o.s.ld : 1}; }

// ---- simple product: 64 x 64 tiles, 4 x 4 sums per thread, any strides -------------------------------------------------------

constexpr int kTile = 64, kDepth = 16;

template <class T>
__device__ __forceinline__ void finish(const Epilogue& e, long long at, int col, float d) {
  float z[1] = {d};
  if (e.bias) z[0] += to_float(static_cast<const T*>(e.bias)[col]);
  if (e.z) static_cast<T*>(e.z)[at] = held<T>(z[0]);
  activate(z, e.act);
  if (e.residual) z[0] += to_float(static_cast<const T*>(e.residual)[at]);
  static_cast<T*>(e.y)[at] = from_float<T>(z[0]);
}

// Block (x, y): tile, columns fastest, and part y of the sum.  part: partial sums (parts, M, N), or null.
template <class T>
__global__ void __launch_bounds__(kThreads) simple_gemm_kernel(Strided a, Strided b, Gemm g, float* part, long long depth) {
  __shared__ float sa[kDepth][kTile + 4], sb[kDepth][kTile + 4];
  const long long across = (g.N + kTile - 1) / kTile, m0 = blockIdx.x / across * kTile, n0 = blockIdx.x % across * kTile;
  const long long k0 = (long long)blockIdx.y * depth, k1 = min(g.K, k0 + depth);
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  float d[4][4] = {};
  const T *A = static_cast<const T*>(a.base), *B = static_cast<const T*>(b.base);
  for (long long k = k0; k < k1; k += kDepth) {
    for (int e = threadIdx.x; e < kTile * kDepth; e += kThreads) {
      // the index that is dense in memory runs fastest over the threads
      const int ia = a.sk == 1 ? e / kDepth : e % kTile, ka = a.sk == 1 ? e % kDepth : e / kTile;
      const int ib = b.sk == 1 ? e / kDepth : e % kTile, kb = b.sk == 1 ? e % kDepth : e / kTile;
      sa[ka][ia] = m0 + ia < g.M && k + ka < k1 ? to_float(A[(m0 + ia) * a.si + (k + ka) * a.sk]) : 0.f;
      sb[kb][ib] = n0 + ib < g.N && k + kb < k1 ? to_float(B[(n0 + ib) * b.si + (k + kb) * b.sk]) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < kDepth; q++) {
      float u[4], v[4];
#pragma unroll
      for (int i = 0; i < 4; i++) u[i] = sa[q][ty * 4 + i], v[i] = sb[q][tx * 4 + i];
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) d[i][j] += u[i] * v[j];
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
long long simple_workspace(long long M, long long N, long long K) {
  const Split s = split_of(M, N, K);
  return s.parts > 1 ? s.parts * M * N * 4 : 0;
}

template <class T>
int launch_simple_as(const Gemm& g, float* part, const Split& s, unsigned tiles, cudaStream_t stream) {
  simple_gemm_kernel<T><<<dim3(tiles, s.parts), kThreads, 0, stream>>>(strided(g.a), strided(g.b), g, part, s.depth);
  const int st = launched("linear");
  return st != GELIB_OK || !part ? st : launch_join(g, part, s.parts, stream);
}

int launch_simple(const Gemm& g, void* workspace, cudaStream_t stream) {
  if (takes_rows(g)) return launch_rows(g, stream);
  const Split s = split_of(g.M, g.N, g.K);
  float* part = s.parts > 1 ? (float*)workspace : nullptr;
  const long long tiles = ((g.N + kTile - 1) / kTile) * ((g.M + kTile - 1) / kTile);
  if (tiles > 0x7fffffffLL) return fail(GELIB_INVALID, "linear", "too many elements");
  return g.type == GELIB_F32 ? launch_simple_as<float>(g, part, s, (unsigned)tiles, stream)
         : g.type == GELIB_BF16 ? launch_simple_as<__nv_bfloat16>(g, part, s, (unsigned)tiles, stream)
                                : launch_simple_as<__half>(g, part, s, (unsigned)tiles, stream);
}

// ---- gz = gy act'(z) and its column sums ------------------------------------------------------------------------------------------

// Block (x, y): `wide` accesses of V columns, piece y of the rows.  gz.base may be null (not wanted), sums too.
template <class T, int V>
__global__ void __launch_bounds__(kThreads) act_back_kernel(Stored gz, float* sums, const T* gy, const T* z, long long M, int N, int act, int wide, long long per) {
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
      }
      if (gz.base) {
        if (sizeof(T) == 4 && gz.planes == 3) {
          union { __nv_bfloat16 t[V]; typename Raw<V * 2>::type raw; } w[3];
#pragma unroll
          for (int j = 0; j < V; j++) {
            __nv_bfloat16 p[3];
            split3(g[j], p);
            w[0].t[j] = p[0], w[1].t[j] = p[1], w[2].t[j] = p[2];
          }
#pragma unroll
          for (int i = 0; i < 3; i++)
            *reinterpret_cast<typename Raw<V * 2>::type*>((__nv_bfloat16*)gz.base + i * gz.plane + r * gz.ld + c) = w[i].raw;
        } else {
          store_vec<T, V>((T*)gz.base + r * gz.ld + c, g);
        }
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
int launch_act_back(const Stored& gz, float* sums, const gelib_linear_args& p, const Pieces& q, cudaStream_t stream) {
  constexpr int kWide = 16 / sizeof(T);
  const auto kernel = q.V > 1 ? act_back_kernel<T, kWide> : act_back_kernel<T, 1>;
  kernel<<<dim3(q.chunks, q.parts), kThreads, 0, stream>>>(gz, sums, (const T*)p.gy, (const T*)p.z, p.m, p.n, p.act, q.wide, q.per);
  return launched("linear_back");
}

long long up(long long bytes) { return (bytes + 255) / 256 * 256; }

// Which product a layer's call takes: the tensor cores from `kTcWork` multiplications on, which is where their operands' copies (float, or
// rows off their 16-byte boundaries) and a longer start are made up for.
constexpr double kTcWork = 4e6;
bool takes_tc(long long m, long long k, long long n) { return k > 0 && m > 16 && (double)m * k * n >= kTcWork && device_has_tcgen05(); }

Stored x_of(const gelib_linear_args& p) { return {p.x, p.m, p.k, p.ldx, 0, 1}; }
Stored w_of(const gelib_linear_args& p) { return {p.w, p.w_transposed ? p.n : p.k, p.w_transposed ? p.k : p.n, p.ldw, 0, 1}; }

// Bytes that an operand's copy takes, 0 where it is used as it lies.
long long copy_bytes(const Stored& s, int type) { return tc_ready(s, type) ? 0 : up(planes_bytes(s.rows, s.cols, type)); }

long long sums_bytes(const gelib_linear_args& p) {
  return up(4LL * p.n * std::max(pieces_of(p.m, p.n, p.type, false).parts, pieces_of(p.m, p.n, p.type, true).parts));
}

// Puts copies of those that need one behind each other at `at`, by one launch.
int ready(Stored** of, int count, int type, char*& at, cudaStream_t stream) {
  Stored from[3], to[3];
  int n = 0;
  for (int i = 0; i < count; i++) {
    if (tc_ready(*of[i], type)) continue;
    from[n] = *of[i];
    to[n] = planes_of(*of[i], type, at);
    at += up(planes_bytes(of[i]->rows, of[i]->cols, type));
    *of[i] = to[n++];
  }
  return launch_planes(from, to, n, type, stream);
}

}  // namespace

int launch_join(const Gemm& g, const float* part, int parts, cudaStream_t stream) {
  const unsigned blocks = (unsigned)std::min((g.M * g.N + kThreads - 1) / kThreads, 1LL << 20);
  if (g.type == GELIB_F32) join_kernel<float><<<blocks, kThreads, 0, stream>>>(g.e, part, parts, g.M, (int)g.N);
  else if (g.type == GELIB_BF16) join_kernel<__nv_bfloat16><<<blocks, kThreads, 0, stream>>>(g.e, part, parts, g.M, (int)g.N);
  else join_kernel<__half><<<blocks, kThreads, 0, stream>>>(g.e, part, parts, g.M, (int)g.N);
  return launched("linear");
}

long long linear_workspace(const gelib_linear_args& p, bool backward) {
  if (p.m == 0 || p.n == 0) return 0;
  const bool tc = takes_tc(p.m, p.k, p.n);
  const auto gemm = [&](long long M, long long N, long long K) { return tc ? tc_gemm_workspace(M, N, K, p.type) : simple_workspace(M, N, K); };
  const long long copies = tc ? copy_bytes(x_of(p), p.type) + copy_bytes(w_of(p), p.type) : 0;
  if (!backward) return copies + gemm(p.m, p.n, p.k);
  const long long gz = up(planes_bytes(p.m, p.n, p.type));
  return gz + copies + sums_bytes(p) + std::max(gemm(p.m, p.k, p.n), p.w_transposed ? gemm(p.n, p.k, p.m) : gemm(p.k, p.n, p.m));
}

int launch_linear(const gelib_linear_args& p, void* workspace, cudaStream_t stream) {
  Gemm g;
  Stored x = x_of(p), w = w_of(p);
  const bool tc = takes_tc(p.m, p.k, p.n);
  char* at = (char*)workspace;
  if (tc) {
    Stored* both[2] = {&x, &w};
    const int st = ready(both, 2, p.type, at, stream);
    if (st != GELIB_OK) return st;
  }
  g.a = {x, false};
  g.b = {w, !p.w_transposed};
  g.e = {p.y, p.z, p.bias, p.residual, p.act};
  g.M = p.m, g.N = p.n, g.K = p.k, g.type = p.type;
  return tc ? launch_tc_gemm(g, at, stream) : launch_simple(g, at, stream);
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
  const bool tc = takes_tc(p.m, p.k, p.n), products = (p.gx || p.gw) && p.k;
  char* at = (char*)workspace;
  float* sums = (float*)at;
  at += sums_bytes(p);
  // gz: gy as it lies, or written (as the tensor cores want it) by the pass that also sums its columns
  Stored gz = {p.gy, p.m, p.n, p.n, 0, 1}, out = {nullptr, 0, 0, 0, 0, 0};
  if (products && (p.act != GELIB_ACT_NONE || (tc && !tc_ready(gz, p.type)))) {
    out = tc ? planes_of(gz, p.type, at) : Stored{at, p.m, p.n, p.n, 0, 1};
    gz = out;
    at += up(planes_bytes(p.m, p.n, p.type));
  }
  int st;
  if (out.base || p.gb) {
    const Pieces q = pieces_of(p.m, p.n, p.type, is_aligned(p.gy, 16) && is_aligned(p.z, 16));
    float* s = p.gb ? sums : nullptr;
    st = p.type == GELIB_F32 ? launch_act_back<float>(out, s, p, q, stream)
         : p.type == GELIB_BF16 ? launch_act_back<__nv_bfloat16>(out, s, p, q, stream) : launch_act_back<__half>(out, s, p, q, stream);
    if (st != GELIB_OK) return st;
    if (p.gb && (st = launch_sum_parts(p.gb, nullptr, sums, q.parts, p.n, p.type, stream)) != GELIB_OK) return st;
  }
  if (!products) return GELIB_OK;
  Stored x = x_of(p), w = w_of(p);
  if (tc) {
    Stored* of[2];
    int n = 0;
    if (p.gw) of[n++] = &x;
    if (p.gx) of[n++] = &w;
    if ((st = ready(of, n, p.type, at, stream)) != GELIB_OK) return st;
  }
  Gemm g;
  g.e = {nullptr, nullptr, nullptr, nullptr, GELIB_ACT_NONE};
  g.type = p.type;
  if (p.gx) {
    g.a = {gz, false};
    g.b = {w, p.w_transposed != 0};
    g.e.y = p.gx;
    g.M = p.m, g.N = p.k, g.K = p.n;
    if ((st = tc ? launch_tc_gemm(g, at, stream) : launch_simple(g, at, stream)) != GELIB_OK) return st;
  }
  if (p.gw) {
    // in w's own layout: x^T gz, or its transpose gz^T x
    g.a = {p.w_transposed ? gz : x, true};
    g.b = {p.w_transposed ? x : gz, true};
    g.e.y = p.gw;
    g.M = p.w_transposed ? p.n : p.k, g.N = p.w_transposed ? p.k : p.n, g.K = p.m;
    if ((st = tc ? launch_tc_gemm(g, at, stream) : launch_simple(g, at, stream)) != GELIB_OK) return st;
  }
  return GELIB_OK;
}

}  // namespace gelib_b200
