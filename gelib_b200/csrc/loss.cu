// Losses of the rows of z = x w + bias, without keeping z, and their gradients.
//
//   cross entropy   loss_r = log sum_j exp z_rj - z_rt,                             dz_r = g_r (p_r - e_t)
//   distillation    loss_r = T^2 sum_i q_i (log q_i - z_{r,t_i} / T + log sum_j exp(z_rj / T)),   dz_r = g_r T (p_r - sum_i q_i e_{t_i})
//
// with p_r = softmax(z_r / T), and q the softmax of a teacher's few largest logits; T is 1 for cross entropy, whose q is a one.  Then
// gx = dz w^T, gw = x^T dz, gb = sum of dz's rows.
//
// Forward: a product whose epilogue leaves of every row and tile of columns the largest z and the sum of exp((z - largest) / T), and z where
// the row has an entry (loss_tc.cu); a second kernel joins a row's tiles, a third the rows' losses.  Kept for the backward pass are two numbers a
// row.  Backward: z again, piece by piece of the classes, whose epilogue makes dz of it, and two products with that.
//
// dz is an operand of the tensor cores: in 16 bits it is rounded to them.  float16 has no room for the small shares of a large vocabulary, so there dz is
// 2^14 (p - q), times a row's g over the largest finite g of rows with a loss where rows have their own; the rest of the factors comes after the sums.
//
// Rows without a loss have dz = 0, and their x is read as zero: what stands there, NaN say, must not reach gw.  The forward call looks at such rows of a
// 16-bit x, and where one holds what is no finite number the product for gw takes a copy (65536 x 1280 x 100: 62 of 350 us when x was always copied).
//
// What bounds it: the tensor cores, 2 m k n for the loss and 6 m k n for the gradients, a third of them to have z again, which keeping it would save.
// bfloat16, 4096 x 2048 x 65536: 670 us, and two pieces of 365 + 680 (1590 TFLOP/s), 3.3 to 3.4 ms among passes that follow one another, where the power
// limit brings the clock down (the library's sustained rate makes it 3.25).  4096 x 1280 x 32768 with 64 entries a row: 214, 252, 425; 1100 us.  float32, 1000 x 1280 x
// 8192: 97, 113, 191 beside 2 x 18 for the three planes of x and w; 498 us.  Small calls wait for the host: 64 x 192 x 100 float32 84 us, of which the forward
// call takes the host 16, the backward call 55 (an elementwise product's 37: autograd's hand-over) and the rest what two calls in turn cost over each by itself;
// the kernels take 42.
#include <algorithm>
#include <cmath>

#include "loss.h"
#include "plan.h"
#include "planes.cuh"

namespace gelib_b200 {

namespace {

constexpr int kThreads = 256;

constexpr int kRowBlocks = 148 * 4;   // of a launch over rows, at most

// Buckets of a row's classes: 128 at the most.
int bucket_of(int n) { return (int)((n + 32767LL) / 32768) * 256; }
int buckets_of(int n) { return (n + bucket_of(n) - 1) / bucket_of(n); }

// The state and its bytes; p.state may be null.
State state_of(const gelib_linear_loss_args& p, long long* bytes = nullptr) {
  char* at = (char*)p.state;
  State s = {};
  s.scale = (float*)at, at += 256;
  s.odd = (int*)at, at += up(4 * (1 + kRowBlocks));
  s.lse = (float2*)at, at += up(p.m * 8);
  if (p.teacher) {
    s.ids = (int*)at, at += up(p.m * p.top * 4);
    s.q = (float*)at, at += up(p.m * p.top * 4);
    s.starts = (unsigned short*)at, at += up(p.m * (buckets_of(p.n) + 1) * 2);
  }
  if (bytes) *bytes = at - (char*)p.state;
  return s;
}

Entries entries_of(const gelib_linear_loss_args& p, const State& s) {
  return {p.target, s.ids, s.q, s.starts, p.ignore_index, p.top, p.index_bytes, p.n, bucket_of(p.n), buckets_of(p.n)};
}

// ---- before the products ------------------------------------------------------------------------------------------------------

struct Teacher {
  const void* logits;   // null: none
  int type;
  long long m;
  float c;
};
constexpr int kTeacherRows = kCopyThreads / 32;   // of a block
long long teacher_shared(int top) { return kTeacherRows * top * 12LL; }

__device__ __forceinline__ float logit_at(const Teacher& t, long long i) {
  if (t.type == GELIB_F32) return static_cast<const float*>(t.logits)[i];
  return t.type == GELIB_BF16 ? to_float(static_cast<const __nv_bfloat16*>(t.logits)[i]) : to_float(static_cast<const __half*>(t.logits)[i]);
}

// A warp per row: q = softmax(logits / T) over the entries, in ascending order of their classes, and where its buckets begin.
__device__ __forceinline__ void prepare_row(const State& s, const Entries& e, const Teacher& t, long long row, int* ids, int* sorted, float* share) {
  const int lane = threadIdx.x % 32, top = e.top;
  bool invalid = false, number = true;
  float most = -INFINITY;
  for (int i = lane; i < top; i += 32) {
    const long long id = index_at(e.target, row * top + i, e.index_bytes);
    const float v = id < 0 ? -INFINITY : logit_at(t, row * top + i);
    invalid |= id >= e.n;
    number &= v == v;
    ids[i] = id < 0 || id >= e.n ? kNone : (int)id;
    share[i] = v;
    most = fmaxf(most, v);
  }
  invalid = __any_sync(0xffffffffu, invalid), number = __all_sync(0xffffffffu, number);
#pragma unroll
  for (int d = 16; d; d /= 2) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
  float sum = 0;
  for (int i = lane; i < top; i += 32) {
    // a logit of -infinity is no entry; one of +infinity or NaN leaves no number of the row
    const float q = share[i] == -INFINITY ? 0.f : number ? exp2_of(t.c * (share[i] - most)) : NAN;
    share[i] = q;
    if (q == 0.f) ids[i] = kNone;
    sum += q;
  }
#pragma unroll
  for (int d = 16; d; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  __syncwarp();
  int live = 0;
  for (int i = lane; i < top; i += 32) {
    const int id = ids[i];
    int place = 0;
    for (int j = 0; j < top; j++) place += ids[j] < id || (ids[j] == id && j < i);
    live += id != kNone;
    sorted[place] = id;
    s.ids[row * top + place] = invalid && place == 0 ? kInvalid : id;
    s.q[row * top + place] = id == kNone ? 0.f : share[i] / sum;
  }
  live = invalid ? 0 : __reduce_add_sync(0xffffffffu, live);
  __syncwarp();
  for (int b = lane; b <= e.buckets; b += 32) {
    int low = 0, high = live;   // the first place whose class is in bucket b or above
    while (low < high && b < e.buckets) {
      const int mid = (low + high) / 2;
      if (sorted[mid] < b * e.bucket) low = mid + 1;
      else high = mid;
    }
    s.starts[row * (e.buckets + 1) + b] = (unsigned short)(b < e.buckets ? low : live);
  }
}

// The teacher's rows in the first blocks, the operands' copies in the others.  use_copy, where it is given: the first operand is only copied, and *use_copy
// set, if the forward call found x of a row without a loss to hold what is no finite number (s.odd).
template <class T>
__global__ void __launch_bounds__(kCopyThreads) prepare_kernel(const State s, const Entries e, const Teacher t, int teachers, const __grid_constant__ PlaneJobs jobs,
                                                               const float2* rows_out, int* use_copy) {
  extern __shared__ int shared[];
  let_next_begin();
  if ((int)blockIdx.x >= teachers) {
    long long from = 0;
    if (use_copy) {
      bool odd = false;
      const int found = *s.odd;
      for (int i = threadIdx.x; i < found; i += kCopyThreads) odd |= s.odd[1 + i] != 0;
      const int any = __syncthreads_or(odd);
      if (blockIdx.x == 0 && threadIdx.x == 0) *use_copy = any;
      if (!any) from = jobs.first[1];
    }
    copy_planes<T, true>(jobs, blockIdx.x - teachers, gridDim.x - teachers, rows_out, from);
    return;
  }
  const int warp = threadIdx.x / 32;
  const long long row = (long long)blockIdx.x * kTeacherRows + warp;
  int* mine = shared + warp * e.top * 3;
  if (row < t.m) prepare_row(s, e, t, row, mine, mine + e.top, reinterpret_cast<float*>(mine + 2 * e.top));
}

template <class T>
int launch_prepare_as(const char* fn, const State& s, const Entries& e, const Teacher& t, const PlaneJobs& jobs, const float2* rows_out, int* use_copy, cudaStream_t stream) {
  const long long teachers = t.logits ? (t.m + kTeacherRows - 1) / kTeacherRows : 0;
  const long long blocks = teachers + std::min((jobs.first[jobs.count] + kCopyThreads - 1) / kCopyThreads, 148LL * 8);
  const size_t shared = t.logits ? (size_t)teacher_shared(e.top) : 0;
  if (shared > 48 * 1024) {   // asked for anew each time: it is the device's, and the largest is the same for all
    GELIB_CUDA_TRY(fn, cudaFuncSetAttribute(prepare_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)teacher_shared(GELIB_LOSS_MAX_TOP)));
  }
  return launch_after(fn, false, prepare_kernel<T>, dim3((unsigned)blocks), kCopyThreads, shared, stream, s, e, t, (int)teachers, jobs, rows_out, use_copy);
}
int launch_prepare(const char* fn, const State& s, const Entries& e, const Teacher& t, const PlaneJobs& jobs, const float2* rows_out, int* use_copy, int type,
                   cudaStream_t stream) {
  if (jobs.count == 0 && !t.logits) return GELIB_OK;
  return type == GELIB_F32    ? launch_prepare_as<float>(fn, s, e, t, jobs, rows_out, use_copy, stream)
         : type == GELIB_BF16 ? launch_prepare_as<__nv_bfloat16>(fn, s, e, t, jobs, rows_out, use_copy, stream)
                              : launch_prepare_as<__half>(fn, s, e, t, jobs, rows_out, use_copy, stream);
}

// The largest finite |gy| of rows that have a loss (lse); 1 where that is zero or there is none.  Rows without a loss have no say in how the others are
// scaled, and an infinity in one row leaves the others their scale.
__global__ void __launch_bounds__(1024) most_kernel(const float* gy, const float2* lse, long long m, float* most) {
  __shared__ float of[32];
  float v = 0;
#pragma unroll 8
  for (long long i = threadIdx.x; i < m; i += 1024) {
    const float g = fabsf(gy[i]);
    v = fmaxf(v, g < INFINITY && lse[i].y != INFINITY ? g : 0.f);
  }
#pragma unroll
  for (int d = 16; d; d /= 2) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
  if (threadIdx.x % 32 == 0) of[threadIdx.x / 32] = v;
  __syncthreads();
  if (threadIdx.x) return;
  for (int i = 1; i < 32; i++) v = fmaxf(v, of[i]);
  *most = v > 0.f ? v : 1.f;
}

// ---- rows and their losses ----------------------------------------------------------------------------------------------------

struct RowSum {
  double loss;
  long long count;
};
struct Total {
  int reduction;
  float *loss, *scale;

  __device__ __forceinline__ void put(const RowSum& all) const {
    const double by = reduction == GELIB_LOSS_SUM ? 1.0 : all.count ? 1.0 / (double)all.count : 0.0;
    *loss = (float)(all.loss * by);
    *scale = (float)by;
  }
};
constexpr int kRows = 32, kRowThreads = 32 * kRows, kBatch = 4;
constexpr int kFew = 8;   // tiles and entries of a row that a thread takes by itself

struct Rows {
  Entries e;
  State s;
  const float2* part;      // (parts, M)
  const float* at_entry;   // (M, top)
  int parts;
  long long M;
  float c, temperature;
  Total total;
  RowSum* sums;            // of the blocks, where there are several
  const unsigned short* x; // 16-bit x, or null
  long long ldx;
  int K;
  unsigned exponent;       // all ones in an infinity or NaN of x's type
};

// Whether x of the row holds what is no finite number; asked by a whole warp.
__device__ __forceinline__ bool is_odd(const Rows& a, long long row) {
  bool odd = false;
  for (int k = threadIdx.x % 32; k < a.K; k += 32) odd |= (a.x[row * a.ldx + k] & a.exponent) == a.exponent;
  return __any_sync(0xffffffffu, odd);
}
// What the threads of a block found.
__device__ __forceinline__ void put_odd(const Rows& a, bool odd) {
  const int any = __syncthreads_or(odd);
  if (threadIdx.x) return;
  a.s.odd[1 + blockIdx.x] = any;
  if (blockIdx.x == 0) a.s.odd[0] = gridDim.x;
}

// An entry's share of a row's loss; v: the row's largest z and its sum.
__device__ __forceinline__ float entry_of(const Rows& a, long long row, int first, int k, float2 v) {
  if (first == kInvalid || (k == 0 ? first : a.e.ids[row * a.e.top + k]) == kNone) return 0.f;
  const float q = a.e.q ? a.e.q[row * a.e.top + k] : 1.f, to = (v.x - a.at_entry[row * a.e.top + k]) / a.temperature;
  return q == 1.f ? to : q * (logf(q) + to);
}
// The row's loss, from the sum of its entries' shares.
__device__ __forceinline__ float loss_of(const Rows& a, int first, float d, float2 v) {
  return first == kNone ? 0.f : first == kInvalid ? NAN : a.temperature * a.temperature * (d + logf(v.y));
}
__device__ __forceinline__ void put_row(const Rows& a, long long row, int first, float loss, float2 v) {
  // a row of -infinity alone has no softmax
  a.s.lse[row] = {v.x, first == kNone ? INFINITY : first == kInvalid || v.x == -INFINITY ? NAN : log2f(v.y)};
  if (a.total.reduction == GELIB_LOSS_NONE) a.total.loss[row] = loss;
}

// What the threads of a block have, added in a fixed order: a warp's by halves, then the warps' by one thread.
__device__ __forceinline__ void put_sum(const Rows& a, RowSum mine) {
  __shared__ RowSum of[kRows];
  if (a.total.reduction == GELIB_LOSS_NONE) return;
#pragma unroll
  for (int d = 16; d; d /= 2) mine.loss += __shfl_xor_sync(0xffffffffu, mine.loss, d), mine.count += __shfl_xor_sync(0xffffffffu, mine.count, d);
  if (threadIdx.x % 32 == 0) of[threadIdx.x / 32] = mine;
  __syncthreads();
  if (threadIdx.x) return;
  for (int w = 1; w < (int)blockDim.x / 32; w++) mine.loss += of[w].loss, mine.count += of[w].count;
  if (gridDim.x == 1) a.total.put(mine);
  else a.sums[blockIdx.x] = mine;
}

// A block takes 32 rows at a time: 32 warps share the rows' tiles, a row a lane, then every warp joins one row and adds up its entries.  What there is
// is a few numbers a row, so that a handful of blocks waits for memory and little else: kBatch tiles are asked for at a time.
__global__ void __launch_bounds__(kRowThreads) rows_kernel(const Rows a) {
  __shared__ float2 of[kRows][kRows + 1];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  RowSum mine = {0, 0};
  bool odd = false;
  let_next_begin();
  await_previous();
  for (long long m0 = (long long)blockIdx.x * kRows; m0 < a.M; m0 += (long long)gridDim.x * kRows) {
    const long long m = m0 + lane, row = m0 + warp;
    float2 v = {-INFINITY, 0.f};
    if (m < a.M)
      for (int i = warp; i < a.parts; i += 32 * kBatch) {
        float2 w[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; j++) w[j] = i + 32 * j < a.parts ? a.part[(long long)(i + 32 * j) * a.M + m] : float2{-INFINITY, 0.f};
#pragma unroll
        for (int j = 0; j < kBatch; j++) v = joined(v, w[j], a.c);
      }
    of[warp][lane] = v;
    __syncthreads();
    v = of[lane][warp];
    __syncthreads();
#pragma unroll
    for (int d = 16; d; d /= 2) {
      const float2 w = {__shfl_xor_sync(0xffffffffu, v.x, d), __shfl_xor_sync(0xffffffffu, v.y, d)};
      v = joined(v, w, a.c);
    }
    if (row >= a.M) continue;
    const int first = first_class(a.e, row);
    float d = 0;
    for (int k = lane; k < a.e.top; k += 32) d += entry_of(a, row, first, k, v);
#pragma unroll
    for (int i = 16; i; i /= 2) d += __shfl_xor_sync(0xffffffffu, d, i);
    d = loss_of(a, first, d, v);
    if (lane == 0) {
      put_row(a, row, first, d, v);
      mine.loss += d, mine.count += first != kNone;
    }
    if (first == kNone && a.x) odd |= is_odd(a, row);
  }
  put_odd(a, odd);
  put_sum(a, mine);
}

__device__ __forceinline__ RowSum take_row(const Rows& a, long long row, RowSum sum, int* first) {
  float2 v = {-INFINITY, 0.f};
  for (int i = 0; i < a.parts; i++) v = joined(v, a.part[(long long)i * a.M + row], a.c);
  *first = first_class(a.e, row);
  float d = 0;
  for (int k = 0; k < a.e.top; k++) d += entry_of(a, row, *first, k, v);
  d = loss_of(a, *first, d, v);
  put_row(a, row, *first, d, v);
  return {sum.loss + d, sum.count + (*first != kNone)};
}

// A thread per row, where a row has few tiles and entries: a training step of 262144 rows, 64 channels and 100 classes 410 to 285 us.
__global__ void __launch_bounds__(kThreads) short_rows_kernel(const Rows a) {
  RowSum mine = {0, 0};
  bool odd = false;
  let_next_begin();
  await_previous();
  for (long long row0 = (long long)blockIdx.x * kThreads + threadIdx.x / 32 * 32; row0 < a.M; row0 += (long long)gridDim.x * kThreads) {
    const long long row = row0 + threadIdx.x % 32;
    int first = 0;
    if (row < a.M) mine = take_row(a, row, mine, &first);
    unsigned out = a.x ? __ballot_sync(0xffffffffu, row < a.M && first == kNone) : 0;
    while (out) {
      odd |= is_odd(a, row0 + __ffs(out) - 1);
      out &= out - 1;
    }
  }
  put_odd(a, odd);
  put_sum(a, mine);
}

__global__ void __launch_bounds__(kThreads) total_kernel(const RowSum* sums, int parts, Total total) {
  __shared__ RowSum of[kThreads];
  RowSum v = {0, 0};
  await_previous();
  for (int i = threadIdx.x; i < parts; i += kThreads) v.loss += sums[i].loss, v.count += sums[i].count;
  of[threadIdx.x] = v;
  __syncthreads();
  for (int d = kThreads / 2; d; d /= 2) {
    if (threadIdx.x < d) of[threadIdx.x].loss += of[threadIdx.x + d].loss, of[threadIdx.x].count += of[threadIdx.x + d].count;
    __syncthreads();
  }
  if (threadIdx.x == 0) total.put(of[0]);
}

// ---- host ---------------------------------------------------------------------------------------------------------------------

constexpr double kLog2eD = 1.4426950408889634;
float temperature_of(const gelib_linear_loss_args& p) { return p.teacher ? (float)p.temperature : 1.f; }
float slope_of(const gelib_linear_loss_args& p) { return (float)(kLog2eD / temperature_of(p)); }

Stored x_of(const gelib_linear_loss_args& p) { return {p.x, p.m, p.k, p.ldx, 0, 1}; }
Stored w_of(const gelib_linear_loss_args& p) { return {p.w, p.w_transposed ? p.n : p.k, p.w_transposed ? p.k : p.n, p.ldw, 0, 1}; }

// The classes from `first` on.
Stored classes_of(Stored w, bool transposed, int first, int width, int type) {
  const long long bytes = w.planes == 3 ? 2 : type_bytes(type);
  w.base = (const char*)w.base + first * (transposed ? w.ld : 1) * bytes;
  (transposed ? w.rows : w.cols) = width;
  return w;
}

// Classes of a piece of dz: 256 MB of it, or 2048 classes; a multiple of 256.
int piece_of(const gelib_linear_loss_args& p) {
  const long long fit = (1LL << 28) / (p.m * (p.type == GELIB_F32 ? 6 : 2));
  return (int)std::min<long long>(p.n, std::max(2048LL, fit / 256 * 256));
}

long long groups_of(long long m) { return (m + 31) / 32; }

ForwardProduct forward_of(const gelib_linear_loss_args& p) {
  return {x_of(p), w_of(p), !p.w_transposed, p.bias, p.m, p.n, p.k, p.type, entries_of(p, state_of(p)), slope_of(p), nullptr, nullptr};
}
// Partial sums of a row.
int parts_of(const gelib_linear_loss_args& p) {
  const ForwardProduct f = forward_of(p);
  return takes_few(f) ? few_parts(f) : forward_parts(p.m, p.n, p.k, p.type);
}

// Whether a thread takes a row, and how many blocks: one for a few rows, which then adds them all up without another launch.
bool short_rows(const gelib_linear_loss_args& p, int parts) { return parts <= kFew && p.top <= kFew; }
int row_blocks(const gelib_linear_loss_args& p, int parts) {
  if (short_rows(p, parts)) return p.m <= 2 * kThreads ? 1 : (int)std::min<long long>((p.m + kThreads - 1) / kThreads, kRowBlocks);
  return p.m <= 4 * kRows ? 1 : (int)std::min<long long>((p.m + kRows - 1) / kRows, 148 * 2);
}

int launch_rows(const char* fn, const gelib_linear_loss_args& p, const Rows& rows, int blocks, cudaStream_t stream) {
  const bool few_tiles = short_rows(p, rows.parts);
  return launch_after(fn, true, few_tiles ? short_rows_kernel : rows_kernel, dim3(blocks), few_tiles ? kThreads : kRowThreads, 0, stream, rows);
}

int forward(const gelib_linear_loss_args& p, char* at, cudaStream_t stream) {
  static const char* fn = "linear_loss";
  const State s = state_of(p);
  const Entries e = entries_of(p, s);
  const float c = slope_of(p);
  int st;
  ForwardProduct f = forward_of(p);
  const bool few = takes_few(f);
  PlaneJobs jobs = {};
  if (!few) {
    copy_if_needed(&f.x, p.type, at, &jobs);
    copy_if_needed(&f.w, p.type, at, &jobs);
  }
  if ((st = launch_prepare(fn, s, e, {p.teacher, p.teacher_type, p.m, c}, jobs, nullptr, nullptr, p.type, stream)) != GELIB_OK) return st;
  const bool follows = p.teacher || jobs.count > 0;
  const int parts = parts_of(p), blocks = row_blocks(p, parts);
  f.part = (float2*)at, at += up(8LL * parts * p.m);
  f.at_entry = (float*)at, at += up(4 * p.m * p.top);
  if ((st = few ? launch_few(fn, f, follows, stream) : launch_forward_product(fn, f, follows, stream)) != GELIB_OK) return st;
  const Total total = {p.reduction, (float*)p.loss, s.scale};
  const bool wide = p.type == GELIB_F32;
  const Rows rows = {e, s, f.part, f.at_entry, parts, p.m, c, temperature_of(p), total, (RowSum*)at, wide ? nullptr : (const unsigned short*)p.x, p.ldx, p.k,
                     p.type == GELIB_BF16 ? 0x7f80u : 0x7c00u};
  st = launch_rows(fn, p, rows, blocks, stream);
  if (st != GELIB_OK || p.reduction == GELIB_LOSS_NONE || blocks == 1) return st;
  return launch_after(fn, true, total_kernel, dim3(1), kThreads, 0, stream, (const RowSum*)at, blocks, total);
}

// Where things lie in a backward call's workspace.
struct Room {
  Stored x, w, dz;
  Stored x_copy;   // base null, or what stands for x in gw's product where *use_copy is not zero
  int* use_copy;
  PlaneJobs jobs;
  const float2* rows_out;
  float *sums, *sum, *most;
  char* again;     // of few rows, or null
  char* parts;
  long long bytes;
  int piece;
};

// The forward product of few rows adds in another order than the tensor cores (loss_rows.cu), which make z again.  A share is exp of a difference of z and
// the row's log-sum: where z is in the thousands its last place is some 2^-12, and a class that is certain would have that for a gradient instead of
// nothing.  So the largest z and the log-sum of few rows are made again too, of the z that the gradients have: one more product of a row of tiles, whose
// weights are read once more (a step of 1 x 1280 x 32768: bfloat16 143 to 175 us, float32 362 to 464).
struct Again {
  State s;             // odd and lse are the backward call's own
  ForwardProduct f;
  float* loss;
  long long bytes;
};
Again again_at(const gelib_linear_loss_args& p, const Stored& x, const Stored& w, char* begin) {
  char* at = begin;
  Again a = {state_of(p), forward_of(p)};
  a.s.odd = (int*)at, at += 256;
  a.s.lse = (float2*)at, at += up(8 * p.m);
  a.loss = (float*)at, at += up(4 * p.m);
  a.f.x = x, a.f.w = w;
  a.f.part = (float2*)at, at += up(8LL * forward_parts(p.m, p.n, p.k, p.type) * p.m);
  a.f.at_entry = (float*)at, at += up(4 * p.m * p.top);
  a.bytes = at - begin;
  return a;
}
int launch_again(const char* fn, const gelib_linear_loss_args& p, const Again& a, bool follows, cudaStream_t stream) {
  const int parts = forward_parts(p.m, p.n, p.k, p.type), st = launch_forward_product(fn, a.f, follows, stream);
  if (st != GELIB_OK) return st;
  const Rows rows = {a.f.e, a.s, a.f.part, a.f.at_entry, parts, p.m, a.f.c, temperature_of(p), {GELIB_LOSS_NONE, a.loss, nullptr}, nullptr, nullptr, p.ldx, p.k, 0};
  return launch_rows(fn, p, rows, 1, stream);
}

// What a backward call does with a piece of `width` classes from `first` on; addresses in the workspace where `at` is one.
struct Piece {
  SlopeProduct slope;
  Grads grads;
};
Piece piece_at(const gelib_linear_loss_args& p, const State& s, const Room& r, int first, int width) {
  const Stored &x = r.x, &w = r.w, &dz = r.dz;
  float *sum = r.sum, *most = r.most;
  Piece q = {};
  const bool none = p.reduction == GELIB_LOSS_NONE;
  const float up = p.type == GELIB_F16 ? 16384.f : 1.f;
  const bool t = p.w_transposed != 0;
  SlopeProduct& f = q.slope;
  f.x = x, f.w = classes_of(w, t, first, width, p.type), f.w_by_sum = !t, f.bias = p.bias;
  f.M = p.m, f.N = width, f.K = p.k, f.type = p.type, f.first = first;
  f.e = entries_of(p, s), f.c = slope_of(p), f.up = up, f.lse = s.lse;
  f.gy = none ? (const float*)p.gy : nullptr, f.most = most;
  f.dz = dz;
  f.dz.cols = width;
  Grads& g = q.grads;
  g.type = p.type;
  g.a0 = none ? most : (const float*)p.gy, g.a1 = none ? nullptr : s.scale, g.a2 = temperature_of(p) / up;
  if (p.gx) g.g[g.count++] = {{f.dz, false}, {f.w, t}, p.m, p.k, width, p.gx, p.k, sum, first == 0, first + width == p.n};
  if (p.gw) {   // in w's own layout: x^T dz, or its transpose dz^T x
    const Operand a = {t ? f.dz : x, true}, b = {t ? x : f.dz, true};
    char* y = (char*)p.gw + (long long)first * (t ? p.k : 1) * type_bytes(p.type);
    g.g[g.count++] = {a, b, t ? width : p.k, t ? p.k : width, p.m, y, t ? p.k : p.n, nullptr, true, true, r.x_copy, t};
    g.use_other = r.use_copy;
  }
  return q;
}

Room room_of(const gelib_linear_loss_args& p, char* begin) {
  Room r = {};
  char* at = begin;
  r.piece = piece_of(p);
  r.x = x_of(p), r.w = w_of(p);
  if (p.gw) {   // a copy in which rows without a loss are zero; in 16 bits only where they have to be
    const Stored to = planes_at(r.x, p.type, at);
    r.jobs.add(r.x, to, p.type);
    if (tc_ready(r.x, p.type)) r.x_copy = to, r.use_copy = (int*)at, at += 256;
    else r.x = to;
    r.rows_out = state_of(p).lse;
  } else {
    copy_if_needed(&r.x, p.type, at, &r.jobs);
  }
  copy_if_needed(&r.w, p.type, at, &r.jobs);
  r.dz = planes_at({nullptr, p.m, r.piece, 0, 0, 1}, p.type, at);
  if (p.gb) r.sums = (float*)at, at += up(4 * groups_of(p.m) * r.piece);
  if (p.gx && r.piece < p.n) r.sum = (float*)at, at += up(4LL * p.m * p.k);
  if (p.reduction == GELIB_LOSS_NONE && p.type == GELIB_F16) r.most = (float*)at, at += 256;
  if (takes_few(forward_of(p))) r.again = at, at += again_at(p, r.x, r.w, at).bytes;
  r.parts = at;
  long long most = 0;
  for (int first : {0, (p.n - 1) / r.piece * r.piece})
    most = std::max(most, grads_workspace(piece_at(p, state_of(p), r, first, std::min(r.piece, p.n - first)).grads));
  r.bytes = at - begin + most;
  return r;
}

int backward(const gelib_linear_loss_args& p, char* workspace, cudaStream_t stream) {
  static const char* fn = "linear_loss_back";
  if (!p.gx && !p.gw && !p.gb) return GELIB_OK;
  State s = state_of(p);
  const Room r = room_of(p, workspace);
  int st;
  if (r.most) {
    most_kernel<<<1, 1024, 0, stream>>>((const float*)p.gy, s.lse, p.m, r.most);
    if ((st = launched(fn)) != GELIB_OK) return st;
  }
  if ((st = launch_prepare(fn, s, entries_of(p, s), {}, r.jobs, r.rows_out, r.use_copy, p.type, stream)) != GELIB_OK) return st;
  bool follows = r.jobs.count > 0;
  if (r.again) {
    const Again a = again_at(p, r.x, r.w, r.again);
    if ((st = launch_again(fn, p, a, follows, stream)) != GELIB_OK) return st;
    s.lse = a.s.lse;
    follows = true;
  }
  for (int first = 0; first < p.n; first += r.piece) {
    const int width = std::min(r.piece, p.n - first);
    Piece q = piece_at(p, s, r, first, width);
    q.slope.sums = r.sums;
    if (p.gb) q.grads.sums = r.sums, q.grads.gb = (char*)p.gb + (long long)first * type_bytes(p.type), q.grads.sum_parts = groups_of(p.m), q.grads.sum_n = width;
    if ((st = launch_slope_product(fn, q.slope, follows, stream)) != GELIB_OK) return st;
    if ((st = launch_grads(fn, q.grads, true, r.parts, stream)) != GELIB_OK) return st;
    follows = true;
  }
  return GELIB_OK;
}

}  // namespace

long long linear_loss_state_bytes(const gelib_linear_loss_args& p) {
  long long bytes;
  state_of(p, &bytes);
  return bytes;
}

long long linear_loss_workspace(const gelib_linear_loss_args& p, bool backward) {
  if (backward) return p.gx || p.gw || p.gb ? room_of(p, nullptr).bytes : 0;
  const long long copies = takes_few(forward_of(p)) ? 0 : copy_bytes(x_of(p), p.type) + copy_bytes(w_of(p), p.type);
  const int parts = parts_of(p);
  return copies + up(8LL * parts * p.m) + up(4 * p.m * p.top) +
         up(row_blocks(p, parts) * (long long)sizeof(RowSum));
}

int launch_linear_loss(const gelib_linear_loss_args& p, void* workspace, cudaStream_t stream) {
  if (!device_has_tcgen05()) return fail(GELIB_INVALID, "linear_loss", "the device has no tensor cores of the fifth generation");
  return forward(p, (char*)workspace, stream);
}

int launch_linear_loss_back(const gelib_linear_loss_args& p, void* workspace, cudaStream_t stream) {
  if (!device_has_tcgen05()) return fail(GELIB_INVALID, "linear_loss_back", "the device has no tensor cores of the fifth generation");
  return backward(p, (char*)workspace, stream);
}

}  // namespace gelib_b200
