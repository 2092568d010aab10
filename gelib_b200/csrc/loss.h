// What the losses' kernels share: the sparse side of a row, the state between the two calls, and the products on the tensor cores (loss_tc.cu).
#pragma once
#include <climits>

#include "heads.h"
#include "linear.h"

namespace gelib_b200 {

constexpr int kNone = INT_MAX;   // of a row's sorted classes: no entry
constexpr int kInvalid = -2;     // a row's first class: one of its classes does not exist

// What the forward call leaves for the backward call.
struct State {
  float* scale;   // 1 over the rows that have a loss, or 1
  int* odd;       // how many numbers follow, and whether x of a row without a loss holds what is no finite number, by blocks of rows (16-bit x)
  float2* lse;    // (m) the largest z and log2 sum exp2(c (z - largest)), c = log2(e) / T; their sum by itself would cost digits where z is in the thousands.
                  // The second is infinite where a row has no loss
  int* ids;       // (m, top) with a teacher: the classes of entries with q > 0 in ascending order, then kNone
  float* q;       // (m, top) their q
  unsigned short* starts;   // (m, buckets + 1): the place of a row's first entry of each bucket of classes, and how many there are
};

// The sparse side of a row: its classes and their shares.
struct Entries {
  const void* target;   // without a teacher: class numbers as the caller has them
  const int* ids;       // with one
  const float* q;
  const unsigned short* starts;
  long long ignore;
  int top, index_bytes, n;
  int bucket, buckets;  // classes of a bucket, and how many there are
};

// z = x w + bias of all rows and classes.  Of every row and half of a tile's columns (the half of every other 16) the largest z and the sum of
// exp2(c (z - largest)) go to part (parts, M), z at the row's classes to at_entry (M, top).
struct ForwardProduct {
  Stored x, w;
  bool w_by_sum;
  const void* bias;
  long long M;
  int N, K, type;
  Entries e;
  float c;
  float2* part;
  float* at_entry;
};
int forward_parts(long long M, int N, int K, int type);
int launch_forward_product(const char* fn, const ForwardProduct& p, bool follows, cudaStream_t stream);

// The same for a few rows (loss_rows.cu), of x and w as the caller has them.
bool takes_few(const ForwardProduct& p);
int few_parts(const ForwardProduct& p);
int launch_few(const char* fn, const ForwardProduct& p, bool follows, cudaStream_t stream);

// z again, of the N classes from `first` on, and of it dz = up g (p - q), which the tensor cores take: 16-bit, or three planes.
struct SlopeProduct {
  Stored x, w;          // w: of these classes
  bool w_by_sum;
  const void* bias;
  long long M;
  int N, K, type, first;
  Entries e;
  float c, up;
  const float2* lse;
  const float *gy, *most;   // g of row r is gy[r] / *most; gy null: 1
  Stored dz;
  float* sums;              // (rows / 32, N): sums of dz's columns over 32 rows, or null
};
int launch_slope_product(const char* fn, const SlopeProduct& p, bool follows, cudaStream_t stream);

// y = *a0 *a1 a2 A B, where the sum over pieces goes through `sum`: to be begun (first), added to, or finished (last).
struct GradProduct {
  Operand a, b;
  long long M, N, K;
  void* y;
  long long ldy;
  float* sum;     // (M, N), or null: one piece
  bool first, last;
  Stored other;          // base null, or what stands for b (other_b) or a
  bool other_b;
};
struct Grads {
  GradProduct g[2];
  int count = 0, type;
  const float *a0, *a1;   // either may be null
  float a2;
  const float* sums = nullptr;   // (sum_parts, sum_n): added up, times the same, into gb
  void* gb = nullptr;
  long long sum_parts = 0;
  int sum_n = 0;
  const int* use_other = nullptr;   // not zero: the products' `other` operands are taken
};
long long grads_workspace(const Grads& g);
int launch_grads(const char* fn, const Grads& g, bool follows, void* workspace, cudaStream_t stream);

#ifdef __CUDACC__
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

// A row's classes from `from` on and below `to`, in ascending order, with their shares.  Where they begin and end is looked up by buckets of classes, so that a
// row without any costs two numbers (a search by bisection for every row and tile took the kernel that makes dz from 236 to 295 us with 64 entries a row at
// 4096 x 1280 x 32768); the one after the next is asked for when the next is.
struct Next {
  int cls, after;     // or kNone
  float q, q_after;
  int at, end;        // the next one's place, and behind the last

  __device__ __forceinline__ void look(const Entries& e, long long row, int place, int& c, float& share) {
    c = kNone, share = 0.f;
    if (place < end) c = e.ids[row * e.top + place], share = e.q[row * e.top + place];
  }
  __device__ __forceinline__ void begin(const Entries& e, long long row, bool live, int from, int to) {
    at = 0, end = 0, q = 1.f, after = kNone, q_after = 0.f, cls = kNone;
    if (!live || from >= to) return;
    if (!e.ids) {
      cls = first_class(e, row);
      if (cls < 0 || cls < from || cls >= to) cls = kNone;
      return;
    }
    const unsigned short* starts = e.starts + row * (e.buckets + 1);
    at = starts[from / e.bucket], end = starts[(to - 1) / e.bucket + 1];
    look(e, row, at, cls, q);
    look(e, row, at + 1, after, q_after);
    while (cls < from) advance(e, row);
  }
  __device__ __forceinline__ void advance(const Entries& e, long long row) {
    at++;
    cls = after, q = q_after;
    if (cls != kNone) look(e, row, at + 1, after, q_after);
  }
};
#endif

}  // namespace gelib_b200
