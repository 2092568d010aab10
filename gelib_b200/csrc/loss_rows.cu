// The forward product of a loss for at most eight rows: one object at a time is scored, and what counts is how fast the weights come in.
//
// The weights are read once, as they lie and in whatever type.  Where a row of them holds all k of one class, a warp owns classes, four at a time, and its
// lanes share k; where it holds all classes of one k, a lane owns 16 bytes' worth of classes and the warps of a block share k.  Of the rows' z only
// the largest, the sum of exp2(c (z - largest)) over a block's classes and z at the rows' entries are kept, as by the tensor cores (loss_tc.cu).
//
// A backward call of few rows makes their log-sums again on the tensor cores, whose z its gradients have (loss.cu).
//
// One row of 1280 bfloat16 over 32768 classes, weights from memory: 21 us for 84 MB (4.0 TB/s; 65536 classes 4.5), 27 with the join of the rows; by the tensor cores,
// whose tiles of 128 rows would be empty but for one, 29 and 35.  Which rows are few, in us a call, 1280 x 32768, here and there: bfloat16 two rows 26 and 30, four 43
// and 33, eight 57 and 33.  float32, whose planes need not be made, one 42 and 163, eight 68 and 163: eight rows are what these kernels hold in registers, and
// the times would cross at more.
#include <algorithm>

#include "loss.h"

namespace gelib_b200 {

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kAcrossThreads = 512, kAcrossWarps = kAcrossThreads / 32;
constexpr int kSms = 148;
constexpr int blocks_of_sm(int rows) { return rows == 1 ? 4 : rows == 2 ? 3 : 2; }   // that its registers have room for

struct RowsArgs {
  const void *x, *w, *bias;
  long long ldx, ldw;
  int M, N, K;
  Entries e;
  float c;
  float2* part;
  float* at_entry;
  int per;      // classes of a warp (rows of weights per class), or of a block
};

template <class T, int V>
__device__ __forceinline__ void load_x(const T* x, bool wide, float (&v)[V]) {
  if constexpr (V > 1) {
    if (wide) {
      load_vec<T, V>(x, v);
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < V; j++) v[j] = to_float(x[j]);
}

// z of one class joins what a lane has of its row.
__device__ __forceinline__ void take(const RowsArgs& a, float z, int cls, int row, Next& next, float2& sum) {
  while (next.cls <= cls) {
    if (next.cls == cls) a.at_entry[row * a.e.top + next.at] = z;
    next.advance(a.e, row);
  }
  sum = joined(sum, {z, z == -INFINITY ? 0.f : 1.f}, a.c);
}

// Partial sums of a block's warps, (warp, row), to the block's part.
template <int kCount>
__device__ __forceinline__ void join_warps(const RowsArgs& a, const float2 (&of)[kCount][8]) {
  __syncthreads();
  if ((int)threadIdx.x < a.M) {
    float2 s = of[0][threadIdx.x];
#pragma unroll
    for (int w = 1; w < kCount; w++) s = joined(s, of[w][threadIdx.x], a.c);
    a.part[(long long)blockIdx.x * a.M + threadIdx.x] = s;
  }
}

// w (N, K): a warp's classes are a.per that follow one another; lane 4 r + j of it keeps the sums of row r over every fourth.
template <class T, int V, int M>
__global__ void __launch_bounds__(kThreads, blocks_of_sm(M)) along_kernel(const RowsArgs a) {
  __shared__ float2 of[kWarps][8];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, row = lane / 4;
  const long long c0 = ((long long)blockIdx.x * kWarps + warp) * a.per, c1 = min((long long)a.N, c0 + a.per);
  const T *x = static_cast<const T*>(a.x), *w = static_cast<const T*>(a.w);
  const bool wide = a.M == 1 || a.ldx % V == 0;
  let_next_begin();
  await_previous();
  Next next;
  next.begin(a.e, row, row < a.M && c0 < c1, (int)c0, (int)c1);
  float2 sum = {-INFINITY, 0.f};
  for (long long c = c0; c < c1; c += 4) {
    float s[M][4];
#pragma unroll
    for (int m = 0; m < M; m++)
#pragma unroll
      for (int j = 0; j < 4; j++) s[m][j] = 0;
    const T* of_class[4];
#pragma unroll
    for (int j = 0; j < 4; j++) of_class[j] = w + min(c + j, c1 - 1) * a.ldw;
#pragma unroll 2
    for (int k = lane * V; k < a.K; k += 32 * V) {
      float u[4][V];
#pragma unroll
      for (int j = 0; j < 4; j++) load_vec<T, V>(of_class[j] + k, u[j]);
#pragma unroll
      for (int m = 0; m < M; m++) {
        float v[V];
        load_x<T, V>(x + min(m, a.M - 1) * a.ldx + k, wide, v);
#pragma unroll
        for (int j = 0; j < 4; j++) s[m][j] += dot_of(u[j], v);
      }
    }
    float z = 0;
#pragma unroll
    for (int m = 0; m < M; m++)
#pragma unroll
      for (int j = 0; j < 4; j++) {
#pragma unroll
        for (int d = 16; d; d /= 2) s[m][j] += __shfl_xor_sync(0xffffffffu, s[m][j], d);
        if (lane == 4 * m + j) z = s[m][j];
      }
    const long long cls = c + lane % 4;
    if (row < a.M && cls < c1) {
      if (a.bias) z += to_float(static_cast<const T*>(a.bias)[cls]);
      take(a, z, (int)cls, row, next, sum);
    }
    __syncwarp();
  }
#pragma unroll
  for (int d = 1; d < 4; d *= 2) {
    const float2 o = {__shfl_xor_sync(0xffffffffu, sum.x, d), __shfl_xor_sync(0xffffffffu, sum.y, d)};
    sum = joined(sum, o, a.c);
  }
  if (lane % 4 == 0) of[warp][row] = sum;
  join_warps(a, of);
}

// w (K, N): a block's classes are 32 V that follow one another; its warps take every sixteenth k, and their sums meet in shared memory row by row.
template <class T, int V, int M>
__global__ void __launch_bounds__(kAcrossThreads) across_kernel(const RowsArgs a) {
  __shared__ float2 of[8][8];
  __shared__ float sums[kAcrossWarps][32 * V + 1];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, n0 = blockIdx.x * 32 * V, n = n0 + lane * V;
  const T *x = static_cast<const T*>(a.x), *w = static_cast<const T*>(a.w);
  let_next_begin();
  await_previous();
  float s[M][V];
#pragma unroll
  for (int m = 0; m < M; m++)
#pragma unroll
    for (int j = 0; j < V; j++) s[m][j] = 0;
  if (n < a.N)
#pragma unroll 8
    for (int k = warp; k < a.K; k += kAcrossWarps) {
      float u[V];
      load_vec<T, V>(w + k * a.ldw + n, u);
#pragma unroll
      for (int m = 0; m < M; m++) fma_all(s[m], u, to_float(x[min(m, a.M - 1) * a.ldx + k]), s[m]);
    }
#pragma unroll
  for (int m = 0; m < M; m++) {
    if (m >= a.M) break;
#pragma unroll
    for (int j = 0; j < V; j++) sums[warp][j * 32 + lane] = s[m][j];
    __syncthreads();
    float2 sum = {-INFINITY, 0.f};
    Next next;
    const int at = (int)threadIdx.x, cls = n0 + at;   // class `at` of the block lies at [at % V][at / V]
    next.begin(a.e, m, at < 32 * V && cls < a.N, cls, cls + 1);
    if (at < 32 * V && cls < a.N) {
      float z = a.bias ? to_float(static_cast<const T*>(a.bias)[cls]) : 0.f;
#pragma unroll
      for (int q = 0; q < kAcrossWarps; q++) z += sums[q][at % V * 32 + at / V];
      take(a, z, cls, m, next, sum);
    }
    __syncwarp();
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const float2 o = {__shfl_xor_sync(0xffffffffu, sum.x, d), __shfl_xor_sync(0xffffffffu, sum.y, d)};
      sum = joined(sum, o, a.c);
    }
    if (lane == 0 && warp < 8) of[warp][m] = sum;   // 256 classes at the most
    __syncthreads();
  }
  join_warps(a, of);
}

// How many classes of a lane, or numbers of one class, go in one access: 16 bytes of them or one; where a row has all classes also 8 or 4 bytes, so that
// few classes make more blocks.
int width_of(const ForwardProduct& p) {
  const auto fits = [&](int V) {
    return is_aligned(p.w.base, V * type_bytes(p.type)) && (p.w_by_sum ? p.N : p.K) % V == 0 && (p.w.ld % V == 0 || p.w.rows <= 1) &&
           (p.w_by_sum || is_aligned(p.x.base, 16));
  };
  int V = 16 / type_bytes(p.type);
  if (!p.w_by_sum) return fits(V) ? V : 1;
  while (V > 1 && (!fits(V) || (p.N + 32 * V - 1) / (32 * V) < kSms)) V /= 2;
  return V;
}
int blocks_of(const ForwardProduct& p, int* per) {
  if (p.w_by_sum) {
    *per = 32 * width_of(p);
    return (p.N + *per - 1) / *per;
  }
  const long long warps = kSms * blocks_of_sm((int)p.M) * kWarps;   // of one round
  *per = (int)std::max(4LL, (p.N + warps - 1) / warps);
  return (int)((p.N + (long long)*per * kWarps - 1) / ((long long)*per * kWarps));
}

template <class T, int V, int M>
int launch_rows_as(const char* fn, const RowsArgs& a, bool along, int blocks, bool follows, cudaStream_t stream) {
  if (along) {
    if constexpr (V == 1 || V * sizeof(T) == 16) return launch_after(fn, follows, along_kernel<T, V, M>, dim3(blocks), kThreads, 0, stream, a);
  }
  return launch_after(fn, follows, across_kernel<T, V, M>, dim3(blocks), kAcrossThreads, 0, stream, a);
}
template <class T, int V>
int launch_rows_of(const char* fn, const RowsArgs& a, bool along, int blocks, bool follows, cudaStream_t stream) {
  if (a.M == 1) return launch_rows_as<T, V, 1>(fn, a, along, blocks, follows, stream);
  if (a.M == 2) return launch_rows_as<T, V, 2>(fn, a, along, blocks, follows, stream);
  if constexpr (sizeof(T) == 4) return a.M <= 4 ? launch_rows_as<T, V, 4>(fn, a, along, blocks, follows, stream) : launch_rows_as<T, V, 8>(fn, a, along, blocks, follows, stream);
  return fail(GELIB_INVALID, fn, "too many rows");
}
template <class T>
int launch_rows_type(const char* fn, const RowsArgs& a, bool along, int blocks, int V, bool follows, cudaStream_t stream) {
  if constexpr (sizeof(T) == 2)
    if (V == 8) return launch_rows_of<T, 8>(fn, a, along, blocks, follows, stream);
  if (V == 4) return launch_rows_of<T, 4>(fn, a, along, blocks, follows, stream);
  if (V == 2) return launch_rows_of<T, 2>(fn, a, along, blocks, follows, stream);
  return launch_rows_of<T, 1>(fn, a, along, blocks, follows, stream);
}

}  // namespace

// Rows that are few: 16-bit ones by the times above, float32 ones as many as the kernels take.
bool takes_few(const ForwardProduct& p) { return p.M <= (p.type == GELIB_F32 ? 8 : 2); }

int few_parts(const ForwardProduct& p) {
  int per;
  return blocks_of(p, &per);
}

int launch_few(const char* fn, const ForwardProduct& p, bool follows, cudaStream_t stream) {
  RowsArgs a = {p.x.base, p.w.base, p.bias, p.x.ld, p.w.ld, (int)p.M, p.N, p.K, p.e, p.c, p.part, p.at_entry, 0};
  const int blocks = blocks_of(p, &a.per), V = width_of(p);
  const bool along = !p.w_by_sum;
  return p.type == GELIB_F32    ? launch_rows_type<float>(fn, a, along, blocks, V, follows, stream)
         : p.type == GELIB_BF16 ? launch_rows_type<__nv_bfloat16>(fn, a, along, blocks, V, follows, stream) : launch_rows_type<__half>(fn, a, along, blocks, V, follows, stream);
}

}  // namespace gelib_b200
