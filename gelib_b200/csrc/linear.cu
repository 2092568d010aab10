// A dense layer with its epilogue, and its gradients:
//
//   z = x w + bias,  y = act(z) + residual
//   gz = gy act'(z),  gx = gz w^T,  gw = x^T gz,  gb = sum of gz's rows
//
// In 16 bits gz = gy act'(z) is rounded to the type it has as an operand of the matrix instructions, as the output is once more: a gradient is off by
// the root of two times the output's own rounding (2.4e-3 of its norm against 1.7e-3 in bfloat16).  Eight rows and fewer take no matrix
// instructions, and gz stays in float.
//
// Forward is one matrix product whose epilogue adds, activates and rounds once.  Backward is one pass over gy and z for gz and the
// column sums, and two products.  Sums over rows are split over blocks when there are few tiles, as partial sums that are added
// in a fixed order.
//
// The tensor cores (gemm_tc.cu) do the products of nine rows and more, at most eight go to linear_rows.cu, and a simple product of any layout does what
// is left.  A backward call is three launches: what goes before the products (one pass over gy and z beside the operands'
// copies), both products, and the joins of partial sums beside the bias's gradient.  With gradients, us a pass of the Python call: 777 x
// 204 x 131 bfloat16 86 and 1000 x 1280 x 512 float32 87, of which autograd's own hand-over is about 50; 65536 x 112 x 112 float32 with
// a residual 131: copies 13 and 27, whose bytes the operator could do without, products 41 and 42, where a tile's two slabs, sums and results follow one
// another (tensor cores 17 and 32 %, DRAM 25 %); 4096 x 7168 x 2048 bfloat16 326, the products 260 (tensor cores 80 and 91 %).
#include <algorithm>

#include "readout.h"
#include "linear.h"
#include "plan.h"
#include "planes.cuh"

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

// Block (x, y): tile, columns fastest, and part y of the sum.  part: partial sums (parts, M, N), or null.  TA, TB: the operands' types, T or float.
template <class T, class TA, class TB>
__global__ void __launch_bounds__(kThreads) simple_gemm_kernel(Strided a, Strided b, Gemm g, float* part, long long depth) {
  __shared__ float sa[kDepth][kTile + 4], sb[kDepth][kTile + 4];
  const long long across = (g.N + kTile - 1) / kTile, m0 = blockIdx.x / across * kTile, n0 = blockIdx.x % across * kTile;
  const long long k0 = (long long)blockIdx.y * depth, k1 = min(g.K, k0 + depth);
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  float d[4][4] = {};
  const TA* A = static_cast<const TA*>(a.base);
  const TB* B = static_cast<const TB*>(b.base);
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

// The partial sums added up in their order, and the epilogue; columns' sums in the last blocks.  A block has 32 accesses side by side and eight
// threads for each, which share the parts where there are many; their sums are added in a fixed order.
struct JoinArgs {
  Joins joins;
  long long blocks[3];   // of the two joins and of the sums
};

template <class T, int V>
__device__ __forceinline__ void join_block(const Joins::Join& a, long long block, float (&t)[8][32][5]) {
  const int lane = threadIdx.x % 32, group = threadIdx.x / 32;
  const bool shared = a.parts >= 16;
  const long long at = shared ? (block * 32 + lane) * V : (block * kThreads + threadIdx.x) * V;
  float d[V];
#pragma unroll
  for (int j = 0; j < V; j++) d[j] = 0;
  if (at < a.size) {
    const int step = shared ? 8 : 1;
#pragma unroll 4
    for (int i = shared ? group : 0; i < a.parts; i += step) {
      float v[V];
      load_vec<float, V>(a.part + i * a.size + at, v);
#pragma unroll
      for (int j = 0; j < V; j++) d[j] += v[j];
    }
  }
  if (shared) {
#pragma unroll
    for (int j = 0; j < V; j++) t[group][lane][j] = d[j];
    __syncthreads();
    if (group > 0) return;
#pragma unroll
    for (int j = 0; j < V; j++) {
      d[j] = 0;
#pragma unroll
      for (int i = 0; i < 8; i++) d[j] += t[i][lane][j];
    }
  }
  if (at < a.size)
#pragma unroll
    for (int j = 0; j < V; j++) finish<T>(a.e, at + j, (int)((at + j) % a.N), d[j]);
}

template <class T>
__global__ void __launch_bounds__(kThreads) join_kernel(const __grid_constant__ JoinArgs a) {
  __shared__ float t[8][32][5];
  await_previous();
  long long block = blockIdx.x;
#pragma unroll
  for (int i = 0; i < 2; i++) {
    if (block < a.blocks[i]) {
      if (a.joins.j[i].vec) join_block<T, 4>(a.joins.j[i], block, t);
      else join_block<T, 1>(a.joins.j[i], block, t);
      return;
    }
    block -= a.blocks[i];
  }
  // eight columns, 32 threads for each
  float* sums = &t[0][0][0];
  const int lane = threadIdx.x % 8, group = threadIdx.x / 8, n = a.joins.sum_n;
  const long long c = block * 8 + lane;
  float s = 0;
  if (c < n)
#pragma unroll 4
    for (int i = group; i < a.joins.sum_parts; i += 32) s += a.joins.sums[(long long)i * n + c];
  sums[threadIdx.x] = s;
  __syncthreads();
  if (group == 0 && c < n) {
    s = 0;
#pragma unroll
    for (int i = 0; i < 32; i++) s += sums[i * 8 + lane];
    static_cast<T*>(a.joins.gb)[c] = from_float<T>(s);
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
long long simple_workspace(const Gemm& g) {
  if (takes_rows(g)) return 0;
  const Split s = split_of(g.M, g.N, g.K);
  return s.parts > 1 ? (s.parts * g.M * g.N * 4 + 255) / 256 * 256 : 0;
}

int launch_simple(const Gemm& g, void* workspace, Joins* joins, cudaStream_t stream) {
  if (takes_rows(g)) return launch_rows(g, stream);
  const Split s = split_of(g.M, g.N, g.K);
  float* part = s.parts > 1 ? (float*)workspace : nullptr;
  if (part) joins->add(g, part, s.parts);
  const long long tiles = ((g.N + kTile - 1) / kTile) * ((g.M + kTile - 1) / kTile);
  if (tiles > 0x7fffffffLL) return fail(GELIB_INVALID, "linear", "too many elements");
  const dim3 grid((unsigned)tiles, s.parts);
  const Strided a = strided(g.a), b = strided(g.b);
  const auto run = [&](auto kernel) { kernel<<<grid, kThreads, 0, stream>>>(a, b, g, part, s.depth); };
  const auto run_type = [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    if (g.a.s.in_float) run(simple_gemm_kernel<T, float, T>);
    else if (g.b.s.in_float) run(simple_gemm_kernel<T, T, float>);
    else run(simple_gemm_kernel<T, T, T>);
  };
  if (g.type == GELIB_F32) run(simple_gemm_kernel<float, float, float>);
  else if (g.type == GELIB_BF16) run_type((__nv_bfloat16*)nullptr);
  else run_type((__half*)nullptr);
  return launched("linear");
}

// ---- before the products: gz = gy act'(z) and its column sums, beside the operands' copies ------------------------------------------

struct ActBack {
  Stored gz;              // base null: not wanted
  float* sums;            // (parts, N), or null
  const void *gy, *z;
  long long M, per;       // rows, and of a piece
  int N, act;
  int wide, chunks, parts;   // a block has `wide` accesses side by side; chunks * parts blocks, 0 where there is nothing to do
};

template <class T, int V>
__global__ void __launch_bounds__(kThreads) prepare_kernel(const __grid_constant__ ActBack a, const __grid_constant__ PlaneJobs jobs) {
  __shared__ float chan[kThreads * V];
  let_next_begin();
  const int blocks = a.chunks * a.parts;
  if ((int)blockIdx.x >= blocks) {
    copy_planes<T>(jobs, blockIdx.x - blocks, gridDim.x - blocks);
    return;
  }
  const Stored& gz = a.gz;
  float* sums = a.sums;
  const T *gy = static_cast<const T*>(a.gy), *z = static_cast<const T*>(a.z);
  const long long M = a.M, piece = blockIdx.x / a.chunks;
  const int N = a.N, act = a.act, wide = a.wide, tx = threadIdx.x % wide, ty = threadIdx.x / wide, high = kThreads / wide;
  const int c = ((int)blockIdx.x % a.chunks * wide + tx) * V;
  const long long r1 = min(M, (piece + 1) * a.per);
  float s[V];
#pragma unroll
  for (int j = 0; j < V; j++) s[j] = 0;
  if (ty < high && c < N)
    for (long long r = piece * a.per + ty; r < r1; r += high) {
      float g[V];
      load_vec<T, V>(gy + r * N + c, g);
      if (act != GELIB_ACT_NONE) {
        float q[V];
        load_vec<T, V>(z + r * N + c, q);
        activate_back(g, q, act);
      }
      if (gz.base) {
        if (sizeof(T) == 4 && gz.planes == 3) {
          union { uint32_t t[(V + 1) / 2]; typename Raw<V * 2>::type raw; } w[3];
#pragma unroll
          for (int j = 0; j < V; j += 2) {
            uint32_t p[3];
            split3(g[j], j + 1 < V ? g[j + 1] : 0.f, p);
#pragma unroll
            for (int i = 0; i < 3; i++) w[i].t[j / 2] = p[i];
          }
#pragma unroll
          for (int i = 0; i < 3; i++)
            *reinterpret_cast<typename Raw<V * 2>::type*>((__nv_bfloat16*)gz.base + i * gz.plane + r * gz.ld + c) = w[i].raw;
        } else if (sizeof(T) == 2 && gz.in_float) {
          float* to = (float*)gz.base + r * gz.ld + c;
          if constexpr (V % 4 == 0)
#pragma unroll
            for (int j = 0; j < V; j += 4) *reinterpret_cast<float4*>(to + j) = make_float4(g[j], g[j + 1], g[j + 2], g[j + 3]);
          else
#pragma unroll
            for (int j = 0; j < V; j++) to[j] = g[j];
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
      sums[piece * N + c + j] = t;
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
  const long long parts = std::max(1LL, std::min((M + 4 * high - 1) / (4 * high), (long long)(kSms * 4 + p.chunks - 1) / p.chunks));
  p.per = (M + parts - 1) / parts;
  p.parts = (int)((M + p.per - 1) / p.per);
  return p;
}

template <class T>
int launch_prepare_as(const ActBack& a, int V, const PlaneJobs& jobs, cudaStream_t stream) {
  const long long copies = std::min((jobs.first[jobs.count] + kThreads - 1) / kThreads, (long long)kSms * 8);
  const unsigned blocks = (unsigned)(a.chunks * a.parts + copies);
  if (blocks == 0) return GELIB_OK;
  if (V > 1) prepare_kernel<T, 16 / sizeof(T)><<<blocks, kThreads, 0, stream>>>(a, jobs);
  else prepare_kernel<T, 1><<<blocks, kThreads, 0, stream>>>(a, jobs);
  return launched("linear");
}
int launch_prepare(const ActBack& a, int V, const PlaneJobs& jobs, int type, cudaStream_t stream) {
  return type == GELIB_F32 ? launch_prepare_as<float>(a, V, jobs, stream)
         : type == GELIB_BF16 ? launch_prepare_as<__nv_bfloat16>(a, V, jobs, stream) : launch_prepare_as<__half>(a, V, jobs, stream);
}

Stored x_of(const gelib_linear_args& p);
Stored w_of(const gelib_linear_args& p);

// Whether a layer's call takes the tensor cores.  At most eight rows do not: their forward and the gradient of x read the weights once
// (linear_rows.cu), and the gradient of w is a sum of eight products.  More do, backward always (17 x 8 x 8 to 32 x 1280 x 1280, us: float32 13 to 23
// against 21 to 60 of the simple product, bfloat16 11 to 21 against 27 to 72), forward unless operands have to be copied for less than 40000
// multiplications (72 x 17 x 11 float32 8.7 simple, 11.3 with copies; 20 x 64 x 64 12.6 and 11.2; bfloat16 in place 6.6 whatever the size, 7.9 to 41).
constexpr double kTcCopied = 4e4;
bool takes_tc(const gelib_linear_args& p, bool backward) {
  if (p.m <= 8 || p.k == 0 || !device_has_tcgen05()) return false;
  return backward || (tc_ready(x_of(p), p.type) && tc_ready(w_of(p), p.type)) || (double)p.m * p.k * p.n >= kTcCopied;
}

Stored x_of(const gelib_linear_args& p) { return {p.x, p.m, p.k, p.ldx, 0, 1}; }
Stored w_of(const gelib_linear_args& p) { return {p.w, p.w_transposed ? p.n : p.k, p.w_transposed ? p.k : p.n, p.ldw, 0, 1}; }

// gz = gy act'(z): in the type that the tensor cores take, in float for the other products.
long long gz_bytes(const gelib_linear_args& p, bool tc) { return tc ? planes_bytes(p.m, p.n, p.type) : up(4LL * p.m * p.n); }

long long sums_bytes(const gelib_linear_args& p) {
  return up(4LL * p.n * std::max(pieces_of(p.m, p.n, p.type, false).parts, pieces_of(p.m, p.n, p.type, true).parts));
}

// The forward's product; the backward's, those of them that are wanted, whose operands x, w, gz may be copies.
Gemm forward_of(const gelib_linear_args& p, const Stored& x, const Stored& w) {
  Gemm g = {};
  g.a = {x, false};
  g.b = {w, !p.w_transposed};
  g.e = {p.y, p.z, p.bias, p.residual, p.act};
  g.M = p.m, g.N = p.n, g.K = p.k, g.type = p.type;
  return g;
}
int backward_of(const gelib_linear_args& p, const Stored& x, const Stored& w, const Stored& gz, Gemm (&g)[2]) {
  int count = 0;
  if (p.gx && p.k) {
    Gemm& q = g[count++];
    q = {};
    q.a = {gz, false};
    q.b = {w, p.w_transposed != 0};
    q.e.y = p.gx;
    q.M = p.m, q.N = p.k, q.K = p.n, q.type = p.type;
  }
  if (p.gw && p.k) {   // in w's own layout: x^T gz, or its transpose gz^T x
    Gemm& q = g[count++];
    q = {};
    q.a = {p.w_transposed ? gz : x, true};
    q.b = {p.w_transposed ? x : gz, true};
    q.e.y = p.gw;
    q.M = p.w_transposed ? p.n : p.k, q.N = p.w_transposed ? p.k : p.n, q.K = p.m, q.type = p.type;
  }
  return count;
}

long long products_workspace(const Gemm* g, int count, bool tc) {
  if (tc) return count ? tc_gemm_workspace(g, count) : 0;
  long long bytes = 0;
  for (int i = 0; i < count; i++) bytes += simple_workspace(g[i]);
  return bytes;
}
int launch_products(const Gemm* g, int count, bool tc, bool follows, char* at, Joins* joins, cudaStream_t stream) {
  if (tc) return count ? launch_tc_gemm(g, count, follows, at, joins, stream) : GELIB_OK;
  for (int i = 0; i < count; i++) {
    const int st = launch_simple(g[i], at, joins, stream);
    if (st != GELIB_OK) return st;
    at += simple_workspace(g[i]);
  }
  return GELIB_OK;
}

}  // namespace

void Joins::add(const Gemm& g, const float* part, int parts) {
  const int four = 4 * type_bytes(g.type);
  const bool vec = g.N % 4 == 0 && is_aligned(g.e.y, four);
  j[count++] = {g.e, part, parts, (int)g.N, vec, g.M * g.N};
}

int launch_joins(const Joins& joins, int type, cudaStream_t stream) {
  JoinArgs a = {};
  a.joins = joins;
  long long blocks = 0;
  for (int i = 0; i < joins.count; i++) {
    const Joins::Join& q = joins.j[i];
    const long long each = (long long)(q.parts >= 16 ? 32 : kThreads) * (q.vec ? 4 : 1);
    a.blocks[i] = (q.size + each - 1) / each;
    blocks += a.blocks[i];
  }
  if (joins.gb) blocks += a.blocks[2] = (joins.sum_n + 7) / 8;
  if (blocks == 0) return GELIB_OK;
  if (blocks > 0x7fffffffLL) return fail(GELIB_INVALID, "linear", "too many elements");
  const auto kernel = type == GELIB_F32 ? join_kernel<float> : type == GELIB_BF16 ? join_kernel<__nv_bfloat16> : join_kernel<__half>;
  return launch_after("linear", true, kernel, dim3((unsigned)blocks), kThreads, 0, stream, a);
}

long long linear_workspace(const gelib_linear_args& p, bool backward) {
  if (p.m == 0 || p.n == 0) return 0;
  const bool tc = takes_tc(p, backward);
  const Stored x = x_of(p), w = w_of(p), gz = {p.gy, p.m, p.n, p.n, 0, 1};
  const long long copies = tc ? copy_bytes(x, p.type) + copy_bytes(w, p.type) : 0;
  if (!backward) {
    const Gemm g = forward_of(p, x, w);
    return copies + products_workspace(&g, 1, tc);
  }
  Gemm g[2];
  const int count = backward_of(p, x, w, gz, g);
  return gz_bytes(p, tc) + copies + sums_bytes(p) + products_workspace(g, count, tc);
}

int launch_linear(const gelib_linear_args& p, void* workspace, cudaStream_t stream) {
  Stored x = x_of(p), w = w_of(p);
  const bool tc = takes_tc(p, false);
  char* at = (char*)workspace;
  int st;
  PlaneJobs jobs = {};
  if (tc) {
    copy_if_needed(&x, p.type, at, &jobs);
    copy_if_needed(&w, p.type, at, &jobs);
    if ((st = launch_prepare({}, 1, jobs, p.type, stream)) != GELIB_OK) return st;
  }
  const Gemm g = forward_of(p, x, w);
  Joins joins;
  if ((st = launch_products(&g, 1, tc, jobs.count > 0, at, &joins, stream)) != GELIB_OK) return st;
  return launch_joins(joins, p.type, stream);
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
  const bool tc = takes_tc(p, true), products = (p.gx || p.gw) && p.k;
  char* at = (char*)workspace;
  Joins joins;
  if (p.gb) {
    joins.sums = (float*)at;
    joins.gb = p.gb;
    joins.sum_n = p.n;
    at += sums_bytes(p);
  }
  // gz: gy as it lies, or written (as the tensor cores want it) by the pass that also sums its columns
  Stored gz = {p.gy, p.m, p.n, p.n, 0, 1}, x = x_of(p), w = w_of(p);
  ActBack back = {};
  PlaneJobs jobs = {};
  if (products && (p.act != GELIB_ACT_NONE || (tc && !tc_ready(gz, p.type)))) {
    if (tc) gz = planes_at(gz, p.type, at);
    else {
      gz.base = at;
      gz.in_float = true;
      at += gz_bytes(p, tc);
    }
    back.gz = gz;
  }
  if (tc && p.gw) copy_if_needed(&x, p.type, at, &jobs);
  if (tc && p.gx) copy_if_needed(&w, p.type, at, &jobs);
  const Pieces q = pieces_of(p.m, p.n, p.type, is_aligned(p.gy, 16) && is_aligned(p.z, 16));
  if (back.gz.base || p.gb) {
    back.sums = (float*)joins.sums;
    back.gy = p.gy, back.z = p.z, back.M = p.m, back.N = p.n, back.act = p.act;
    back.per = q.per, back.wide = q.wide, back.chunks = q.chunks, back.parts = q.parts;
    joins.sum_parts = q.parts;
  }
  int st = launch_prepare(back, q.V, jobs, p.type, stream);
  if (st != GELIB_OK) return st;
  Gemm g[2];
  const int count = backward_of(p, x, w, gz, g);
  if ((st = launch_products(g, count, tc, jobs.count > 0 || back.chunks > 0, at, &joins, stream)) != GELIB_OK) return st;
  return launch_joins(joins, p.type, stream);
}

}  // namespace gelib_b200
