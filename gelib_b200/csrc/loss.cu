// Losses of the rows of z = x w + bias, without keeping z, and their gradients.
//
//   cross entropy   loss_r = log sum_j exp z_rj - z_rt,                             dz_r = g_r (p_r - e_t)
//   distillation    loss_r = T^2 sum_i q_i (log q_i - z_{r,t_i} / T + log sum_j exp(z_rj / T)),   dz_r = g_r T (p_r - sum_i q_i e_{t_i})
//
// with p_r = softmax(z_r / T), and q the softmax of a teacher's few largest logits; T is 1 for cross entropy, whose q is a one.  Then
// gx = dz w^T, gw = x^T dz, gb = sum of dz's rows.
//
// Forward: a product whose epilogue leaves of every row and tile of columns the largest z and the sum of exp((z - largest) / T), and z where
// the teacher has an entry; a second kernel joins a row's tiles, a third the rows' losses.  Kept for the backward pass is the logarithm of the sum,
// one number a row.  Backward: z again, piece by piece of the columns, whose epilogue makes dz of it, and two products with that.
#include <algorithm>
#include <cfloat>
#include <climits>
#include <cmath>

#include "heads.h"
#include "plan.h"

namespace gelib_b200 {

namespace {

constexpr int kThreads = 256;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kNone = INT_MAX;   // of a row's sorted classes: no entry
constexpr int kInvalid = -2;     // a row's first class: one of its classes does not exist

// What the forward call leaves for the backward call.
struct State {
  float* scale;   // 1 over the rows that have a loss, or 1
  float2* lse;    // (m) the largest z and log2 sum exp2(c (z - largest)), c = log2(e) / T; their sum by itself would cost digits where z is in the thousands.
                  // The second is infinite where a row has no loss
  int* ids;       // (m, top) with a teacher: the classes of entries with q > 0 in ascending order, then kNone
  float* q;       // (m, top) their q
};
long long up(long long bytes) { return (bytes + 255) / 256 * 256; }
State state_of(const gelib_linear_loss_args& p) {
  char* at = (char*)p.state;
  State s;
  s.scale = (float*)at, at += 256;
  s.lse = (float2*)at, at += up(p.m * 8);
  s.ids = (int*)at, at += up(p.m * p.top * 4);
  s.q = (float*)at;
  return s;
}

// The sparse side of a row: its classes and their shares.
struct Entries {
  const void* target;   // without a teacher: class numbers as the caller has them
  const int* ids;       // with one
  const float* q;
  long long ignore;
  int top, index_bytes, n;
};
Entries entries_of(const gelib_linear_loss_args& p, const State& s) {
  return {p.target, p.teacher ? s.ids : nullptr, p.teacher ? s.q : nullptr, p.ignore_index, p.top, p.index_bytes, p.n};
}
// The row's first class: kNone where it has no loss, kInvalid where it is not one of the n.
__device__ __forceinline__ int first_class(const Entries& e, long long row) {
  if (e.ids) return e.ids[row * e.top];
  const long long t = index_at(e.target, row, e.index_bytes);
  return t == e.ignore ? kNone : t < 0 || t >= e.n ? kInvalid : (int)t;
}

__device__ __forceinline__ float exp2_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The sum of exp2(c z) over some columns as (largest z, sum of exp2(c (z - largest))).  No columns, or only -infinity: (-infinity, 0).
__device__ __forceinline__ float2 joined(float2 a, float2 b, float c) {
  const float top = fmaxf(a.x, b.x), from = top == -INFINITY ? 0.f : top;
  // fmaxf drops a NaN, the sums keep it
  return {top, a.y * exp2_of(c * (a.x - from)) + b.y * exp2_of(c * (b.x - from))};
}

// ---- the teacher -------------------------------------------------------------------------------------------------------------

// A warp per row: q = softmax(logits / T) over the entries, in ascending order of their classes.
template <class T>
__global__ void __launch_bounds__(128) teacher_kernel(State s, Entries e, const T* logits, long long m, float c) {
  __shared__ int ids[4][GELIB_LOSS_MAX_TOP];
  __shared__ float share[4][GELIB_LOSS_MAX_TOP];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, top = e.top;
  const long long row = (long long)blockIdx.x * 4 + warp;
  if (row >= m) return;
  bool invalid = false, number = true;
  float most = -INFINITY;
  for (int i = lane; i < top; i += 32) {
    const long long id = index_at(e.target, row * top + i, e.index_bytes);
    const float t = id < 0 ? -INFINITY : to_float(logits[row * top + i]);
    invalid |= id >= e.n;
    number &= t == t;
    ids[warp][i] = id < 0 || id >= e.n ? kNone : (int)id;
    share[warp][i] = t;
    most = fmaxf(most, t);
  }
  invalid = __any_sync(0xffffffffu, invalid), number = __all_sync(0xffffffffu, number);
#pragma unroll
  for (int d = 16; d; d /= 2) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
  float sum = 0;
  for (int i = lane; i < top; i += 32) {
    // a logit of -infinity is no entry; one of +infinity or NaN leaves no number of the row
    const float q = share[warp][i] == -INFINITY ? 0.f : number ? exp2_of(c * (share[warp][i] - most)) : NAN;
    share[warp][i] = q;
    if (q == 0.f) ids[warp][i] = kNone;
    sum += q;
  }
#pragma unroll
  for (int d = 16; d; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  __syncwarp();
  for (int i = lane; i < top; i += 32) {
    const int id = ids[warp][i];
    int place = 0;
    for (int j = 0; j < top; j++) place += ids[warp][j] < id || (ids[warp][j] == id && j < i);
    s.ids[row * top + place] = invalid && place == 0 ? kInvalid : id;
    s.q[row * top + place] = id == kNone ? 0.f : share[warp][i] / sum;
  }
}

// ---- products -----------------------------------------------------------------------------------------------------------------

// Element (i, k) of an operand at base[i * si + k * sk], i the row of A or the column of B.
struct Strided {
  const void* base;
  long long si, sk;
};

struct Forward {
  float2* part;      // (tiles of columns, M): sums of a row over a tile
  float* at_entry;   // (M, top): z at the row's classes
};
struct Slope {
  float* dz;          // (M, N) of the piece
  float* sums;        // (tiles of rows, N): sums of dz's columns, or null
  const float2* lse;
  const float* gy;    // (M), or null: 1
};
struct Product {
  float* sum;          // (M, N) in float that the product is added to, or null
  void* y;             // the result, element (i, j) at i * si + j * sj, or null: more is to be added
  long long si, sj;
  const float2* skip;  // State's lse: numbers k of the sum whose row has no loss are left out
  bool first;          // nothing has been added to `sum`
  const float *a0, *a1;
  float a2;            // the result is *a0 *a1 a2 times the sum; either may be null
};

constexpr int kTile = 64, kDepth = 16;

// d = A B of a 64 x 64 tile, 4 x 4 sums a thread.
template <class TA, class TB>
__device__ __forceinline__ void tile_product(float (&d)[4][4], const Strided& a, const Strided& b, long long M, long long N, long long K, long long m0, long long n0,
                                             const float2* skip) {
  __shared__ float sa[kDepth][kTile + 4], sb[kDepth][kTile + 4];
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  const TA* A = static_cast<const TA*>(a.base);
  const TB* B = static_cast<const TB*>(b.base);
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) d[i][j] = 0;
  for (long long k = 0; k < K; k += kDepth) {
    for (int e = threadIdx.x; e < kTile * kDepth; e += kThreads) {
      // the index that is dense in memory runs fastest over the threads
      const int ia = a.sk == 1 ? e / kDepth : e % kTile, ka = a.sk == 1 ? e % kDepth : e / kTile;
      const int ib = b.sk == 1 ? e / kDepth : e % kTile, kb = b.sk == 1 ? e % kDepth : e / kTile;
      sa[ka][ia] = m0 + ia < M && k + ka < K && !(skip && skip[k + ka].y == INFINITY) ? to_float(A[(m0 + ia) * a.si + (k + ka) * a.sk]) : 0.f;
      sb[kb][ib] = n0 + ib < N && k + kb < K ? to_float(B[(n0 + ib) * b.si + (k + kb) * b.sk]) : 0.f;
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
}

// z of a tile of rows and of the columns from n0 on of all e.n; c: log2(e) / T.
template <class T>
__device__ __forceinline__ void logits_tile(float (&z)[4][4], const Strided& x, const Strided& w, const T* bias, long long M, int N, int K, long long m0, long long n0) {
  tile_product<T, T>(z, x, w, M, N, K, m0, n0, nullptr);
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const long long n = n0 + threadIdx.x % 16 * 4 + j;
    const float b = bias && n < N ? to_float(bias[n]) : 0.f;
#pragma unroll
    for (int i = 0; i < 4; i++) z[i][j] += b;
  }
}

template <class T>
__global__ void __launch_bounds__(kThreads) forward_kernel(Strided x, Strided w, const T* bias, long long M, int K, Entries e, Forward f, float c) {
  const long long across = (e.n + kTile - 1) / kTile, m0 = blockIdx.x / across * kTile, tile = blockIdx.x % across, n0 = tile * kTile;
  float z[4][4];
  logits_tile(z, x, w, bias, M, e.n, K, m0, n0);
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const long long m = m0 + ty * 4 + i;
    float2 s = {-INFINITY, 0.f};
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (n0 + tx * 4 + j < e.n) s = joined(s, {z[i][j], z[i][j] == -INFINITY ? 0.f : 1.f}, c);
#pragma unroll
    for (int d = 8; d; d /= 2) s = joined(s, {__shfl_xor_sync(0xffffffffu, s.x, d), __shfl_xor_sync(0xffffffffu, s.y, d)}, c);
    if (m >= M) continue;
    if (tx == 0) f.part[tile * M + m] = s;
    const int t = first_class(e, m);
    if (t == kInvalid) continue;
    for (int k = 0; k < e.top; k++) {
      const int col = k == 0 ? t : e.ids[m * e.top + k];
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (n0 + tx * 4 + j == col) f.at_entry[m * e.top + k] = z[i][j];
    }
  }
}

template <class T>
__global__ void __launch_bounds__(kThreads) slope_kernel(Strided x, Strided w, const T* bias, long long M, int K, Entries e, Slope f, float c, int first, int width) {
  __shared__ float sums[16][kTile];
  const long long across = (width + kTile - 1) / kTile, tile_m = blockIdx.x / across, m0 = tile_m * kTile, n0 = first + blockIdx.x % across * kTile;
  float z[4][4];
  logits_tile(z, x, w, bias, M, first + width, K, m0, n0);
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  float s[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const long long m = m0 + ty * 4 + i;
    if (m >= M) continue;
    const float2 lse = f.lse[m];
    const float g = f.gy ? f.gy[m] : 1.f;
    const int t = first_class(e, m);
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const long long n = n0 + tx * 4 + j;
      if (n >= first + width) continue;
      float d = exp2_of(fmaf(c, z[i][j] - lse.x, -lse.y));
      for (int k = 0; k < e.top; k++)
        if ((k == 0 ? t : e.ids[m * e.top + k]) == n) d -= e.q ? e.q[m * e.top + k] : 1.f;
      d = lse.y == INFINITY ? 0.f : d * g;
      s[j] += d;
      f.dz[m * width + (n - first)] = d;
    }
  }
  if (!f.sums) return;
#pragma unroll
  for (int j = 0; j < 4; j++) sums[ty][tx * 4 + j] = s[j];
  __syncthreads();
  if (threadIdx.x < kTile && n0 + threadIdx.x < first + width) {
    float v = 0;
    for (int i = 0; i < 16; i++) v += sums[i][threadIdx.x];
    f.sums[tile_m * width + (n0 - first) + threadIdx.x] = v;
  }
}

template <class T, class TA, class TB>
__global__ void __launch_bounds__(kThreads) product_kernel(Strided a, Strided b, long long M, long long N, long long K, Product p) {
  const long long across = (N + kTile - 1) / kTile, m0 = blockIdx.x / across * kTile, n0 = blockIdx.x % across * kTile;
  float d[4][4];
  tile_product<TA, TB>(d, a, b, M, N, K, m0, n0, p.skip);
  const float scale = p.a2 * (p.a0 ? *p.a0 : 1.f) * (p.a1 ? *p.a1 : 1.f);
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const long long m = m0 + threadIdx.x / 16 * 4 + i, n = n0 + threadIdx.x % 16 * 4 + j;
      if (m >= M || n >= N) continue;
      float v = d[i][j];
      if (p.sum && !p.first) v += p.sum[m * N + n];
      if (p.y) static_cast<T*>(p.y)[m * p.si + n * p.sj] = from_float<T>(v * scale);
      else p.sum[m * N + n] = v;
    }
}

template <class T>
__global__ void __launch_bounds__(kThreads) bias_kernel(T* gb, const float* sums, int parts, int n, const float* a0, const float* a1, float a2) {
  const int c = blockIdx.x * kThreads + threadIdx.x;
  if (c >= n) return;
  float s = 0;
  for (int i = 0; i < parts; i++) s += sums[(long long)i * n + c];
  gb[c] = from_float<T>(s * (a2 * (a0 ? *a0 : 1.f) * (a1 ? *a1 : 1.f)));
}

// ---- rows and their losses ----------------------------------------------------------------------------------------------------

struct RowSum {
  double loss;
  long long count;
};
constexpr int kRows = 32, kGroups = kThreads / kRows;

// A block takes 32 rows; eight groups of lanes share a row's tiles, then a warp takes four rows' entries.
__global__ void __launch_bounds__(kThreads) rows_kernel(Entries e, State s, Forward f, int parts, long long M, float c, float temperature, int reduction, float* loss,
                                                        RowSum* sums) {
  __shared__ float2 of[kGroups][kRows];
  __shared__ float losses[kRows];
  __shared__ int counts[kRows];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const long long m0 = (long long)blockIdx.x * kRows, m = m0 + lane;
  float2 v = {-INFINITY, 0.f};
  if (m < M)
    for (int i = warp; i < parts; i += kGroups) v = joined(v, f.part[(long long)i * M + m], c);
  of[warp][lane] = v;
  __syncthreads();
  for (int r = warp; r < kRows; r += kGroups) {
    const long long row = m0 + r;
    if (row >= M) {
      if (lane == 0) losses[r] = 0, counts[r] = 0;
      continue;
    }
    float2 sum = of[0][r];
    for (int i = 1; i < kGroups; i++) sum = joined(sum, of[i][r], c);
    const int t = first_class(e, row);
    float d = 0;
    for (int k = lane; k < e.top; k += 32) {
      if (t == kInvalid || (k == 0 ? t : e.ids[row * e.top + k]) == kNone) continue;
      const float q = e.q ? e.q[row * e.top + k] : 1.f, to = (sum.x - f.at_entry[row * e.top + k]) / temperature;
      d += q == 1.f ? to : q * (logf(q) + to);
    }
#pragma unroll
    for (int i = 16; i; i /= 2) d += __shfl_xor_sync(0xffffffffu, d, i);
    if (lane) continue;
    d = t == kNone ? 0.f : t == kInvalid ? NAN : temperature * temperature * (d + logf(sum.y));
    // a row of -infinity alone has no softmax
    s.lse[row] = {sum.x, t == kNone ? INFINITY : t == kInvalid || sum.x == -INFINITY ? NAN : log2f(sum.y)};
    if (reduction == GELIB_LOSS_NONE) loss[row] = d;
    losses[r] = d, counts[r] = t != kNone;
  }
  __syncthreads();
  if (reduction == GELIB_LOSS_NONE || threadIdx.x) return;
  RowSum all = {0, 0};
  for (int r = 0; r < kRows; r++) all.loss += losses[r], all.count += counts[r];
  sums[blockIdx.x] = all;
}

__global__ void __launch_bounds__(kThreads) total_kernel(const RowSum* sums, int parts, int reduction, float* loss, float* scale) {
  __shared__ RowSum of[kThreads];
  RowSum v = {0, 0};
  for (int i = threadIdx.x; i < parts; i += kThreads) v.loss += sums[i].loss, v.count += sums[i].count;
  of[threadIdx.x] = v;
  __syncthreads();
  for (int d = kThreads / 2; d; d /= 2) {
    if (threadIdx.x < d) of[threadIdx.x].loss += of[threadIdx.x + d].loss, of[threadIdx.x].count += of[threadIdx.x + d].count;
    __syncthreads();
  }
  if (threadIdx.x) return;
  const double by = reduction == GELIB_LOSS_SUM ? 1.0 : of[0].count ? 1.0 / (double)of[0].count : 0.0;
  *loss = (float)(of[0].loss * by);
  *scale = (float)by;
}

// ---- host ---------------------------------------------------------------------------------------------------------------------

constexpr double kLog2eD = 1.4426950408889634;
float temperature_of(const gelib_linear_loss_args& p) { return p.teacher ? (float)p.temperature : 1.f; }
float slope_of(const gelib_linear_loss_args& p) { return (float)(kLog2eD / temperature_of(p)); }

Strided x_of(const gelib_linear_loss_args& p) { return {p.x, p.ldx, 1}; }
Strided w_of(const gelib_linear_loss_args& p) { return {p.w, p.w_transposed ? p.ldw : 1, p.w_transposed ? 1 : p.ldw}; }

// Columns of a piece of dz: 2^27 numbers, or 2048 columns.
int piece_of(const gelib_linear_loss_args& p) { return (int)std::min<long long>(p.n, std::max(2048LL, ((1LL << 27) / p.m + 255) / 256 * 256)); }

long long tiles(long long n) { return (n + kTile - 1) / kTile; }

template <class T>
int forward_as(const gelib_linear_loss_args& p, char* at, cudaStream_t stream) {
  static const char* fn = "linear_loss";
  const State s = state_of(p);
  const Entries e = entries_of(p, s);
  const float c = slope_of(p);
  const int parts = (int)tiles(p.n);
  Forward f;
  f.part = (float2*)at, at += up(8LL * parts * p.m);
  f.at_entry = (float*)at, at += up(4 * p.m * p.top);
  if (p.teacher) {
    const unsigned blocks = (unsigned)((p.m + 3) / 4);
    if (p.teacher_type == GELIB_F32) teacher_kernel<<<blocks, 128, 0, stream>>>(s, e, (const float*)p.teacher, p.m, c);
    else if (p.teacher_type == GELIB_BF16) teacher_kernel<<<blocks, 128, 0, stream>>>(s, e, (const __nv_bfloat16*)p.teacher, p.m, c);
    else teacher_kernel<<<blocks, 128, 0, stream>>>(s, e, (const __half*)p.teacher, p.m, c);
    const int st = launched(fn);
    if (st != GELIB_OK) return st;
  }
  if (tiles(p.m) * parts > 0x7fffffffLL) return fail(GELIB_INVALID, fn, "too many elements");
  forward_kernel<T><<<(unsigned)(tiles(p.m) * parts), kThreads, 0, stream>>>(x_of(p), w_of(p), (const T*)p.bias, p.m, p.k, e, f, c);
  int st = launched(fn);
  if (st != GELIB_OK) return st;
  const int blocks = (int)((p.m + kRows - 1) / kRows);
  rows_kernel<<<blocks, kThreads, 0, stream>>>(e, s, f, parts, p.m, c, temperature_of(p), p.reduction, (float*)p.loss, (RowSum*)at);
  if ((st = launched(fn)) != GELIB_OK || p.reduction == GELIB_LOSS_NONE) return st;
  total_kernel<<<1, kThreads, 0, stream>>>((const RowSum*)at, blocks, p.reduction, (float*)p.loss, s.scale);
  return launched(fn);
}

template <class T>
int backward_as(const gelib_linear_loss_args& p, char* at, cudaStream_t stream) {
  static const char* fn = "linear_loss_back";
  const State s = state_of(p);
  const Entries e = entries_of(p, s);
  const float c = slope_of(p), temperature = temperature_of(p);
  const int piece = piece_of(p);
  Slope f;
  f.dz = (float*)at, at += up(4 * p.m * piece);
  f.sums = p.gb ? (float*)at : nullptr, at += up(4 * tiles(p.m) * piece);
  float* sum = (float*)at;
  f.lse = s.lse;
  f.gy = p.reduction == GELIB_LOSS_NONE ? (const float*)p.gy : nullptr;
  const float *a0 = f.gy ? nullptr : (const float*)p.gy, *a1 = f.gy ? nullptr : s.scale;
  for (int first = 0; first < p.n; first += piece) {
    const int width = std::min(piece, p.n - first);
    if (tiles(p.m) * tiles(width) > 0x7fffffffLL || tiles(p.k) * std::max(tiles(p.m), tiles(width)) > 0x7fffffffLL) return fail(GELIB_INVALID, fn, "too many elements");
    slope_kernel<T><<<(unsigned)(tiles(p.m) * tiles(width)), kThreads, 0, stream>>>(x_of(p), w_of(p), (const T*)p.bias, p.m, p.k, e, f, c, first, width);
    int st = launched(fn);
    if (st != GELIB_OK) return st;
    const Strided dz = {f.dz, width, 1}, dz_t = {f.dz, 1, width}, x_t = {p.x, 1, p.ldx};
    const long long sk = p.w_transposed ? p.ldw : 1, si = p.w_transposed ? 1 : p.ldw;   // of w: along the classes, along k
    if (p.gx) {
      Product o = {piece < p.n ? sum : nullptr, first + width == p.n ? p.gx : nullptr, p.k, 1, nullptr, first == 0, a0, a1, temperature};
      product_kernel<T, float, T><<<(unsigned)(tiles(p.m) * tiles(p.k)), kThreads, 0, stream>>>(dz, {(const T*)p.w + first * sk, si, sk}, p.m, p.k, width, o);
      if ((st = launched(fn)) != GELIB_OK) return st;
    }
    if (p.gw) {
      // dz's rows without a loss are zero, x's may hold anything: the operand whose rows are left out is x
      const Product o = {nullptr, (T*)p.gw + (long long)first * (p.w_transposed ? p.k : 1), p.w_transposed ? 1 : p.n, p.w_transposed ? p.k : 1, s.lse, true, a0, a1,
                         temperature};
      product_kernel<T, T, float><<<(unsigned)(tiles(p.k) * tiles(width)), kThreads, 0, stream>>>(x_t, dz_t, p.k, width, p.m, o);
      if ((st = launched(fn)) != GELIB_OK) return st;
    }
    if (p.gb) {
      bias_kernel<T><<<(width + kThreads - 1) / kThreads, kThreads, 0, stream>>>((T*)p.gb + first, f.sums, (int)tiles(p.m), width, a0, a1, temperature);
      if ((st = launched(fn)) != GELIB_OK) return st;
    }
  }
  return GELIB_OK;
}

}  // namespace

long long linear_loss_state_bytes(const gelib_linear_loss_args& p) { return 256 + up(p.m * 8) + (p.teacher ? 2 * up(p.m * p.top * 4) : 0); }

long long linear_loss_workspace(const gelib_linear_loss_args& p, bool backward) {
  if (!backward) return up(8LL * tiles(p.n) * p.m) + up(4 * p.m * p.top) + up((p.m + kRows - 1) / kRows * (long long)sizeof(RowSum));
  const int piece = piece_of(p);
  return up(4 * p.m * piece) + up(4 * tiles(p.m) * piece) + (p.gx && piece < p.n ? up(4LL * p.m * p.k) : 0);
}

int launch_linear_loss(const gelib_linear_loss_args& p, void* workspace, cudaStream_t stream) {
  return p.type == GELIB_F32 ? forward_as<float>(p, (char*)workspace, stream)
         : p.type == GELIB_BF16 ? forward_as<__nv_bfloat16>(p, (char*)workspace, stream) : forward_as<__half>(p, (char*)workspace, stream);
}

int launch_linear_loss_back(const gelib_linear_loss_args& p, void* workspace, cudaStream_t stream) {
  return p.type == GELIB_F32 ? backward_as<float>(p, (char*)workspace, stream)
         : p.type == GELIB_BF16 ? backward_as<__nv_bfloat16>(p, (char*)workspace, stream) : backward_as<__half>(p, (char*)workspace, stream);
}

}  // namespace gelib_b200
