// The products of the losses on the tensor cores: three epilogues of the kernel in gemm_tc.cuh.
//
//   forward   z = x w + bias; of z only the largest of a row's columns, the sum of exp2(c (z - largest)) and z at the row's classes are kept.
//   slope     z again; dz = up g (exp2(c (z - largest) - log2 sum) - q), the operand of the gradients.
//   gradients dz w^T and x^T dz by one launch, added up over the pieces of the classes in float.
//
// A lane of the epilogue's warps has 16 columns of a row at a time, so that a row's maximum and sum stay in its registers over a tile.  Largest and sum
// are kept apart for every tile: the sum's exponents are of differences, whatever the size of z.
//
// Tensor cores busy (4096 x 2048 x 16384 bfloat16, z in two runs): forward 87 %, slope 80 %, gradients 91 %; with 64 entries a row and sums of 1280 79, 65 and
// 86 %, where the epilogue of a tile takes as long as its products.  float32 (1000 x 1280 x 8192): 73, 63 and 65 %.
#include "loss.h"

#include "gemm_tc.cuh"

namespace gelib_b200 {

namespace {

// Sixteen columns of z from class n on, of `end`: the sums and the bias.
template <class T>
__device__ __forceinline__ void logits_of(float (&v)[kChunk], const uint32_t (&r)[kChunk], const T* bias, bool wide, int n, int end) {
#pragma unroll
  for (int j = 0; j < kChunk; j++) v[j] = __uint_as_float(r[j]);
  if (!bias) return;
  float b[kChunk];
  if (wide && n + kChunk <= end) {
    constexpr int V = 16 / sizeof(T);
#pragma unroll
    for (int j = 0; j < kChunk; j += V) {
      float w[V];
      load_vec<T, V>(bias + n + j, w);
#pragma unroll
      for (int k = 0; k < V; k++) b[j + k] = w[k];
    }
  } else {
#pragma unroll
    for (int j = 0; j < kChunk; j++) b[j] = n + j < end ? to_float(bias[n + j]) : 0.f;
  }
  add_all(v, v, b);
}

struct ForwardProblem : TcShape {
  const void* bias;
  int wide;          // the bias begins on a 16-byte boundary
  Entries e;
  float c;
  float2* part;
  float* at_entry;
};

template <class T>
struct ForwardEnd {
  using Problem = ForwardProblem;
  static constexpr bool kTwo = false, kBefore = false;
  float2 sum;
  Next next;
  long long row;
  int tile;

  template <int kChunks>
  __device__ __forceinline__ void ahead(const Problem& g, const Item& it, long long m0, int n0, int lane, bool second) {
    row = m0 + lane;
    tile = it.n * 2 + second;
    sum = {-INFINITY, 0.f};
    next.begin(g.e, row, row < g.M, n0, min(g.N, it.n * g.bn + g.bn));
  }
  __device__ __forceinline__ void take(const Problem& g, int, int n, int, uint32_t, const uint32_t (&r)[kChunk], bool) {
    float v[kChunk];
    logits_of<T>(v, r, static_cast<const T*>(g.bias), g.wide, n, g.N);
    if (n + kChunk > g.N)
#pragma unroll
      for (int j = 0; j < kChunk; j++)
        if (n + j >= g.N) v[j] = -INFINITY;
    while (next.cls < n + kChunk) {
      if (next.cls >= n) {
        float z = 0;
#pragma unroll
        for (int j = 0; j < kChunk; j++)
          if (next.cls == n + j) z = v[j];
        g.at_entry[row * g.e.top + next.at] = z;
      }
      next.advance(g.e, row);
    }
    __syncwarp();   // the next read of tensor memory is the whole warp's
    float top = v[0];
#pragma unroll
    for (int j = 1; j < kChunk; j++) top = fmaxf(top, v[j]);
    top = fmaxf(top, sum.x);
    const float from = top == -INFINITY ? 0.f : top;
    add_all(v, v, -from);
    mul_all(v, v, g.c);
#pragma unroll
    for (int j = 0; j < kChunk; j++) v[j] = exp2_of(v[j]);
    sum.y = fmaf(sum.y, exp2_of(g.c * (sum.x - from)), sum_of(v));
    sum.x = top;
  }
  __device__ __forceinline__ void end(const Problem& g, int) {
    if (row < g.M) g.part[(long long)tile * g.M + row] = sum;
  }
};

struct SlopeProblem : TcShape {
  const void* bias;  // of the piece's classes
  int wide;
  Entries e;
  float c, up;
  const float2* lse;
  const float *gy, *most;
  void* dz;
  long long ld, plane;
  float* sums;
  int first;
};

__device__ __forceinline__ void take_from_shared(uint32_t at, float x) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  asm volatile("st.shared.f32 [%0], %1;" ::"r"(at), "f"(v - x) : "memory");
}

template <class T>
struct SlopeEnd {
  using Problem = SlopeProblem;
  static constexpr bool kTwo = false, kBefore = false;
  Next next;
  long long m0;
  float2 lse;
  float g_up;
  bool out, some_out;   // the lane's row has no loss; one of the warp's has none

  template <int kChunks>
  __device__ __forceinline__ void ahead(const Problem& g, const Item& it, long long m, int n0, int lane, bool) {
    m0 = m;
    const long long row = m0 + lane;
    lse = row < g.M ? g.lse[row] : float2{0.f, INFINITY};
    out = lse.y == INFINITY;
    some_out = __any_sync(0xffffffffu, out);
    g_up = g.up;
    if (g.gy && row < g.M) g_up *= g.most ? g.gy[row] / *g.most : g.gy[row];
    next.begin(g.e, row, !out, g.first + n0, g.first + min(g.N, it.n * g.bn + g.bn));
  }
  __device__ __forceinline__ void take(const Problem& g, int, int n, int lane, uint32_t block, const uint32_t (&r)[kChunk], bool) {
    float v[kChunk];
    logits_of<T>(v, r, static_cast<const T*>(g.bias), g.wide, n, g.N);
    add_all(v, v, -lse.x);
    fma_all(v, v, g.c, -lse.y);
#pragma unroll
    for (int j = 0; j < kChunk; j++) v[j] = exp2_of(v[j]);
    mul_all(v, v, g_up);
    if (some_out)
#pragma unroll
      for (int j = 0; j < kChunk; j++) v[j] = out ? 0.f : v[j];
    __syncwarp();
#pragma unroll
    for (int j = 0; j < kAcross; j++)
      tc::sts128(block + (lane * kPitch + 4 * j) * 4, __float_as_uint(v[4 * j]), __float_as_uint(v[4 * j + 1]), __float_as_uint(v[4 * j + 2]), __float_as_uint(v[4 * j + 3]));
    const int cls = g.first + n;
    while (next.cls < cls + kChunk) {
      const long long row = m0 + lane;
      if (next.cls >= cls) take_from_shared(block + (lane * kPitch + next.cls - cls) * 4, g_up * next.q);
      next.advance(g.e, row);
    }
    __syncwarp();
    const int col = lane % kAcross * 4, live = min(4, g.N - n - col);
    const long long m = m0 + lane / kAcross;
    float d[kPasses][4];
#pragma unroll
    for (int pass = 0; pass < kPasses; pass++) {
      const float4 f = tc::lds128(block + ((pass * kRows + lane / kAcross) * kPitch + col) * 4);
      d[pass][0] = f.x, d[pass][1] = f.y, d[pass][2] = f.z, d[pass][3] = f.w;
    }
    if (live > 0) {
      const long long at = m * g.ld + n + col, step = kRows * g.ld;   // rows have room for a multiple of eight
#pragma unroll
      for (int pass = 0; pass < kPasses; pass++) {
        if (m + pass * kRows >= g.M) break;
        if constexpr (sizeof(T) == 4) {
          uint32_t p[3], q[3];
          split3(d[pass][0], d[pass][1], p);
          split3(d[pass][2], d[pass][3], q);
#pragma unroll
          for (int i = 0; i < 3; i++)
            *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(g.dz) + i * g.plane + at + pass * step) = make_uint2(p[i], q[i]);
        } else {
          store_vec<T, 4>(static_cast<T*>(g.dz) + at + pass * step, d[pass]);
        }
      }
    }
    __syncwarp();
    if (!g.sums) return;
    float s[4] = {0, 0, 0, 0};
#pragma unroll
    for (int pass = 0; pass < kPasses; pass++) add_all(s, s, d[pass]);   // rows that are not there are zero
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
      for (int o = kAcross; o < 32; o *= 2) s[j] += __shfl_xor_sync(0xffffffffu, s[j], o);
    if (lane < kAcross && m0 < g.M) {
      float* to = g.sums + m0 / 32 * g.N + n + col;
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (j < live) to[j] = s[j];
    }
  }
  __device__ __forceinline__ void end(const Problem&, int) {}
};

struct GradProblem : TcShape {
  float* part;            // partial sums (splits, M, N), or null
  float* sum;
  void* y;                // null: not finished yet
  long long ldy;
  int begun;              // something has been added to `sum`
  int vec_f, vec_y;       // four columns at a time: in `part` and `sum`, in y
  const float *a0, *a1;
  float a2;
  const float* sums;      // of the launch's first problem: sum_parts rows of sum_n numbers, added up into gb; gb null: not here
  void* gb;
  int sum_parts, sum_n;
};

__device__ __forceinline__ float scale_of(const float* a0, const float* a1, float a2) { return a2 * (a0 ? *a0 : 1.f) * (a1 ? *a1 : 1.f); }

// v (+ what is in `sum`) to y, times `scale`, or to `sum`.
template <class T, int V>
__device__ __forceinline__ void finish_grad(T* y, float* sum, bool begun, float scale, float (&v)[V]) {
  if (sum && begun) {
    float w[V];
    load_vec<float, V>(sum, w);
    add_all(v, v, w);
  }
  if (y) {
    mul_all(v, v, scale);
    store_vec<T, V>(y, v);
  } else {
    store_vec<float, V>(sum, v);
  }
}

template <class T>
struct GradEnd {
  using Problem = GradProblem;
  static constexpr bool kTwo = true, kBefore = true;
  long long m0;
  int split;
  float scale;

  // The bias's gradient, while the first tiles are summed: a column a thread.
  static __device__ __forceinline__ void before(const Problem& g, int thread, int threads) {
    if (!g.gb) return;
    const float scale = scale_of(g.a0, g.a1, g.a2);
    for (int c = thread; c < g.sum_n; c += threads) {
      float s = 0;
#pragma unroll 8
      for (int i = 0; i < g.sum_parts; i++) s += g.sums[(long long)i * g.sum_n + c];
      static_cast<T*>(g.gb)[c] = from_float<T>(s * scale);
    }
    __syncwarp();
  }

  template <int kChunks>
  __device__ __forceinline__ void ahead(const Problem& g, const Item& it, long long m, int, int, bool) {
    m0 = m, split = it.split;
    scale = scale_of(g.a0, g.a1, g.a2);
  }
  __device__ __forceinline__ void take(const Problem& g, int, int n0, int lane, uint32_t block, const uint32_t (&r)[kChunk], bool) {
    __syncwarp();
#pragma unroll
    for (int j = 0; j < kAcross; j++) tc::sts128(block + (lane * kPitch + 4 * j) * 4, r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
    __syncwarp();
    const int col = lane % kAcross * 4, n = n0 + col, live = min(4, g.N - n);
    const long long m = m0 + lane / kAcross;
    float d[kPasses][4];
#pragma unroll
    for (int pass = 0; pass < kPasses; pass++) {
      const float4 f = tc::lds128(block + ((pass * kRows + lane / kAcross) * kPitch + col) * 4);
      d[pass][0] = f.x, d[pass][1] = f.y, d[pass][2] = f.z, d[pass][3] = f.w;
    }
    const bool inside = m0 + 32 <= g.M && n0 + kChunk <= g.N;
    float* sum = g.part ? g.part + (long long)split * g.M * g.N : g.sum;   // partial sums go like those of a first piece
    const bool adds = !g.part && g.begun;
    T* y = g.part ? nullptr : static_cast<T*>(g.y);
    if (inside && (!sum || g.vec_f) && (!y || g.vec_y)) {
      // nothing to be left out: the lane's four accesses one after the other
      if (sum) sum += m * g.N + n;
      const long long step = (long long)kRows * g.N;
      if (sum && adds)
#pragma unroll
        for (int pass = 0; pass < kPasses; pass++) {
          float w[4];
          load_vec<float, 4>(sum + pass * step, w);
          add_all(d[pass], d[pass], w);
        }
      if (y) {
        y += m * g.ldy + n;
#pragma unroll
        for (int pass = 0; pass < kPasses; pass++) {
          mul_all(d[pass], d[pass], scale);
          store_vec<T, 4>(y + pass * kRows * g.ldy, d[pass]);
        }
      } else {
#pragma unroll
        for (int pass = 0; pass < kPasses; pass++) store_vec<float, 4>(sum + pass * step, d[pass]);
      }
      return;
    }
#pragma unroll
    for (int pass = 0; pass < kPasses; pass++)
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const long long row = m + pass * kRows;
        if (row >= g.M || j >= live) continue;
        float one[1] = {d[pass][j]};
        finish_grad<T, 1>(y ? y + row * g.ldy + n + j : nullptr, sum ? sum + row * g.N + n + j : nullptr, adds, scale, one);
      }
    __syncwarp();
  }
  __device__ __forceinline__ void end(const Problem&, int) {}
};

// Partial sums added up in their order, and columns' sums in the last blocks.
constexpr int kJoinThreads = 256;
struct GradJoins {
  struct Join {
    const float* part;
    float* sum;
    void* y;
    long long ldy, M, blocks;
    int parts, N, begun, vec;
  } j[2];
  const float *a0, *a1;
  float a2;
  const float* sums;
  void* gb;
  long long sum_parts;
  int sum_n;
};

// Many parts are shared by the warps of a block, whose sums are added in a fixed order.
constexpr int kSharedParts = 8;
template <class T, int V>
__device__ __forceinline__ void join_grad(const GradJoins::Join& a, long long block, float scale, float (&t)[8][32][5]) {
  const int lane = threadIdx.x % 32, group = threadIdx.x / 32;
  const bool shared = a.parts >= kSharedParts;
  const long long size = a.M * a.N, at = (shared ? block * 32 + lane : block * kJoinThreads + threadIdx.x) * V;
  float d[V];
#pragma unroll
  for (int j = 0; j < V; j++) d[j] = 0;
  if (at < size)
#pragma unroll 4
    for (int i = shared ? group : 0; i < a.parts; i += shared ? 8 : 1) {
      float v[V];
      load_vec<float, V>(a.part + i * size + at, v);
      add_all(d, d, v);
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
  if (at >= size) return;
  const long long m = at / a.N, n = at - m * a.N;
  finish_grad<T, V>(a.y ? static_cast<T*>(a.y) + m * a.ldy + n : nullptr, a.sum ? a.sum + at : nullptr, a.begun, scale, d);
}

template <class T>
__global__ void __launch_bounds__(kJoinThreads) grad_join_kernel(const __grid_constant__ GradJoins a) {
  __shared__ float t[8][32][5];
  let_next_begin();
  await_previous();
  const float scale = scale_of(a.a0, a.a1, a.a2);
  long long block = blockIdx.x;
#pragma unroll
  for (int i = 0; i < 2; i++) {
    if (block < a.j[i].blocks) {
      if (a.j[i].vec) join_grad<T, 4>(a.j[i], block, scale, t);
      else join_grad<T, 1>(a.j[i], block, scale, t);
      return;
    }
    block -= a.j[i].blocks;
  }
  // eight columns, 32 threads for each
  float* sums = &t[0][0][0];
  const int lane = threadIdx.x % 8, group = threadIdx.x / 8;
  const long long c = block * 8 + lane;
  float s = 0;
  if (c < a.sum_n)
#pragma unroll 4
    for (long long i = group; i < a.sum_parts; i += 32) s += a.sums[i * a.sum_n + c];
  sums[threadIdx.x] = s;
  __syncthreads();
  if (group == 0 && c < a.sum_n) {
    s = 0;
#pragma unroll
    for (int i = 0; i < 32; i++) s += sums[i * 8 + lane];
    static_cast<T*>(a.gb)[c] = from_float<T>(s * scale);
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------------------

// The tensor cores cut every sum off at float's last bit, always to the same side, which over 3271 products of float16 put a loss 2.0e-6 of itself off (the
// products summed in float: 1.5e-8).  A loss is float, so z leaves its accumulator often enough that losses are off by less than 2^-20 (9.5e-7) of themselves
// on average.  That grows with the products that stay together: float16, over 12288 rows of 256 classes, 1024 5.1e-7, 1280 6.2e-7, 1792 8.6e-7, 1920
// 9.3e-7, 1984 9.5e-7, 2048 9.9e-7 (bfloat16 8.1e-7 at 1920).  So up to 1920 stay, and longer sums leave in equal runs of at most that.  Leaving costs the epilogue's time,
// which longer sums hide (a step of 4096 x 32768 classes, bfloat16: 1088 products staying 823 us, in two runs 922; 1280 908 and 984, 1536 1057 and 1111, 1920 1342 and 1372).
// It is done in both passes, since a class that is certain has a gradient of p - 1, which is nothing only where the log-sum comes of the same z (of
// few rows the backward call makes it again).
constexpr int kMostSlabs = 30;

// One product whose sums may not be split.
template <template <class> class E, class Problem>
int launch_whole(const char* fn, const Sizes& z, const Operand& x, const Operand& w, int type, const Problem& more, bool follows, cudaStream_t stream) {
  const Plan plan = plan_of(&z, 1, type, true);
  TcMaps maps = {};
  TcArgs<Problem> a = {};
  a.p[0] = more;
  const int st = shape_of(fn, plan, plan.c[0], z, x, w, type, &a.p[0], &maps.a[0], &maps.b[0]);
  if (st != GELIB_OK) return st;
  a.items = a.p[0].items;
  maps.a[1] = maps.a[0], maps.b[1] = maps.b[0];
  finish_args(&a, plan, type);
  if (type == GELIB_F32) return launch_config<E<float>, 3>(fn, plan.cg, maps, a, follows, stream);
  if (a.p[0].slabs > kMostSlabs) {
    const int runs = (a.p[0].slabs + kMostSlabs - 1) / kMostSlabs;
    a.leave = (a.p[0].slabs + runs - 1) / runs;
    return type == GELIB_BF16 ? launch_config<E<__nv_bfloat16>, 1, true>(fn, plan.cg, maps, a, follows, stream)
                              : launch_config<E<__half>, 1, true>(fn, plan.cg, maps, a, follows, stream);
  }
  if (type == GELIB_BF16) return launch_config<E<__nv_bfloat16>, 1>(fn, plan.cg, maps, a, follows, stream);
  return launch_config<E<__half>, 1>(fn, plan.cg, maps, a, follows, stream);
}

Plan plan_for(const Grads& g, Sizes (&z)[kProblems]) {
  for (int i = 0; i < g.count; i++) z[i] = {g.g[i].M, g.g[i].N, g.g[i].K};
  return plan_of(z, g.count, g.type, false);
}

}  // namespace

int forward_parts(long long M, int N, int K, int type) {
  const Sizes z = {M, N, K};
  const int bn = plan_of(&z, 1, type, true).c[0].bn;
  return 2 * ((N + bn - 1) / bn);
}

int launch_forward_product(const char* fn, const ForwardProduct& p, bool follows, cudaStream_t stream) {
  ForwardProblem g = {};
  g.bias = p.bias, g.wide = is_aligned(p.bias, 16);
  g.e = p.e, g.c = p.c, g.part = p.part, g.at_entry = p.at_entry;
  return launch_whole<ForwardEnd>(fn, {p.M, p.N, p.K}, {p.x, false}, {p.w, p.w_by_sum}, p.type, g, follows, stream);
}

int launch_slope_product(const char* fn, const SlopeProduct& p, bool follows, cudaStream_t stream) {
  SlopeProblem g = {};
  g.bias = p.bias ? (const char*)p.bias + (long long)p.first * type_bytes(p.type) : nullptr;
  g.wide = is_aligned(g.bias, 16);
  g.e = p.e, g.c = p.c, g.up = p.up, g.lse = p.lse, g.gy = p.gy, g.most = p.most;
  g.dz = const_cast<void*>(p.dz.base), g.ld = p.dz.ld, g.plane = p.dz.plane;
  g.sums = p.sums, g.first = p.first;
  return launch_whole<SlopeEnd>(fn, {p.M, p.N, p.K}, {p.x, false}, {p.w, p.w_by_sum}, p.type, g, follows, stream);
}

long long grads_workspace(const Grads& g) {
  if (g.count == 0) return 0;
  Sizes z[kProblems];
  const Plan p = plan_for(g, z);
  long long bytes = 0;
  for (int i = 0; i < g.count; i++)
    if (p.c[i].splits > 1) bytes += (p.c[i].splits * g.g[i].M * g.g[i].N * 4 + 255) / 256 * 256;
  return bytes;
}

// Rows of sums that a thread adds up before its first tile: 32 of them (1024 rows of x) take some 2 us, the launch saved 3.
constexpr long long kShortSum = 32;

int launch_grads(const char* fn, const Grads& q, bool follows, void* workspace, cudaStream_t stream) {
  GradJoins joins = {};
  joins.a0 = q.a0, joins.a1 = q.a1, joins.a2 = q.a2;
  int joined = 0;
  bool bias_done = false;
  if (q.count) {
    Sizes z[kProblems];
    const Plan plan = plan_for(q, z);
    TcMaps maps = {};
    TcArgs<GradProblem> a = {};
    char* at = (char*)workspace;
    const bool other = swapped(plan, z, q.count, q.type);
    for (int i = 0; i < q.count; i++) {
      const GradProduct& g = q.g[i];
      const Config& c = plan.c[i];
      const int k = other ? 1 - i : i;
      GradProblem& p = a.p[k];
      const int st = shape_of(fn, plan, c, z[i], g.a, g.b, q.type, &p, &maps.a[k], &maps.b[k]);
      if (st != GELIB_OK) return st;
      if (g.other.base) {
        const Operand& stands = g.other_b ? g.b : g.a;
        const int rows = stands.by_sum ? 64 : g.other_b ? c.bn / plan.cg : 128;
        if (!encode(&maps.other, g.other, q.type, 64, rows)) return fail(GELIB_CUDA_ERROR, fn, "a tensor map could not be made");
        a.other = q.use_other, a.other_of = k, a.other_b = g.other_b;
      }
      p.sum = g.sum, p.begun = !g.first, p.y = g.last ? g.y : nullptr, p.ldy = g.ldy;
      p.a0 = q.a0, p.a1 = q.a1, p.a2 = q.a2;
      p.vec_f = g.N % 4 == 0;
      p.vec_y = g.N % 4 == 0 && g.ldy % 4 == 0 && is_aligned(g.y, 4 * type_bytes(q.type));
      if (c.splits > 1) {
        p.part = (float*)at;
        at += (c.splits * g.M * g.N * 4 + 255) / 256 * 256;
        GradJoins::Join& j = joins.j[joined++];
        j = {p.part, g.sum, p.y, g.ldy, g.M, 0, c.splits, (int)g.N, p.begun, p.vec_f && (!p.y || p.vec_y)};
        const int side = c.splits >= kSharedParts ? 32 : kJoinThreads;   // accesses of a block
        j.blocks = (g.M * g.N / (j.vec ? 4 : 1) + side - 1) / side;
      }
      a.items += p.items;
    }
    if (q.count == 1) maps.a[1] = maps.a[0], maps.b[1] = maps.b[0];
    finish_args(&a, plan, q.type);
    // the bias's gradient goes along where no other launch is needed and a thread's sum is short
    if (q.gb && !joined && q.sum_parts <= kShortSum) {
      GradProblem& p = a.p[0];
      p.sums = q.sums, p.gb = q.gb, p.sum_parts = (int)q.sum_parts, p.sum_n = q.sum_n;
      bias_done = true;
    }
    const int st = q.type == GELIB_F32    ? launch_config<GradEnd<float>, 3>(fn, plan.cg, maps, a, follows, stream)
                   : q.type == GELIB_BF16 ? launch_config<GradEnd<__nv_bfloat16>, 1>(fn, plan.cg, maps, a, follows, stream)
                                          : launch_config<GradEnd<__half>, 1>(fn, plan.cg, maps, a, follows, stream);
    if (st != GELIB_OK) return st;
  }
  long long blocks = joins.j[0].blocks + joins.j[1].blocks;
  if (q.gb && !bias_done) {
    joins.sums = q.sums, joins.gb = q.gb, joins.sum_parts = q.sum_parts, joins.sum_n = q.sum_n;
    blocks += (q.sum_n + 7) / 8;
  }
  if (blocks == 0) return GELIB_OK;
  if (blocks > 0x7fffffffLL) return fail(GELIB_INVALID, fn, "too many elements");
  const auto kernel = q.type == GELIB_F32 ? grad_join_kernel<float> : q.type == GELIB_BF16 ? grad_join_kernel<__nv_bfloat16> : grad_join_kernel<__half>;
  return launch_after(fn, true, kernel, dim3((unsigned)blocks), kJoinThreads, 0, stream, joins);
}

}  // namespace gelib_b200
