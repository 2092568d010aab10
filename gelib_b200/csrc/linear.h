// Dense layers: what the C ABI hands to the kernels, and the matrix products that they are made of.
#pragma once
#include "common.h"

namespace gelib_b200 {

// What happens to a sum d before it is stored: z = d + bias, y = act(z) + residual; z is stored too where it is asked for.  y, z, residual are dense.
struct Epilogue {
  void* y;
  void* z;                       // or null
  const void *bias, *residual;   // or null
  int act;
};

// A matrix as it lies in memory: rows of dense columns, `ld` elements apart.  planes 3: a float matrix as the sum of three bfloat16
// ones, `plane` elements apart (each holds the next eight bits of the significand).  in_float: it is float although the call's type is another, which
// only the products without tensor cores take.
struct Stored {
  const void* base;
  long long rows, cols, ld, plane;
  int planes;
  bool in_float = false;
};

// One operand of D = A B, M x K or K x N: its rows are the sum's index, or (by_sum false) M's or N's.
struct Operand {
  Stored s;
  bool by_sum;
};

struct Gemm {
  Operand a, b;
  Epilogue e;
  long long M, N, K;
  int type;      // of the result, and of the operands that have one plane
};

// What is left to do after the products of a call, by one launch: partial sums to be joined, and the bias's gradient.
struct Joins {
  struct Join {
    Epilogue e;
    const float* part;     // (parts, M, N)
    int parts, N, vec;
    long long size;        // M N
  } j[2];
  int count = 0;
  const float* sums = nullptr;   // (sum_parts, sum_n): added up into gb
  void* gb = nullptr;
  int sum_parts = 0, sum_n = 0;
  void add(const Gemm& g, const float* part, int parts);
};
int launch_joins(const Joins& joins, int type, cudaStream_t stream);

// Tensor-core products (gemm_tc.cu), one or two of them by one launch.  Operands must be `tc_ready`: three planes of a float matrix, or 16-bit, on 16-byte
// boundaries.
bool tc_ready(const Stored& s, int type);
long long tc_gemm_workspace(const Gemm* g, int count);
// `follows`: the launch before on the stream is one of this call's.
int launch_tc_gemm(const Gemm* g, int count, bool follows, void* workspace, Joins* joins, cudaStream_t stream);

// Products of at most eight rows (linear_rows.cu).
bool takes_rows(const Gemm& g);
int launch_rows(const Gemm& g, cudaStream_t stream);

long long linear_workspace(const gelib_linear_args& p, bool backward);
int launch_linear(const gelib_linear_args& p, void* workspace, cudaStream_t stream);
int launch_linear_back(const gelib_linear_args& p, void* workspace, cudaStream_t stream);

#ifdef __CUDACC__
template <class T>
__device__ __forceinline__ T held(float z) {   // z as it is kept for the backward pass: an infinity would have no derivative
  if constexpr (std::is_same_v<T, __half>) z = z < -65504.f ? -65504.f : z > 65504.f ? 65504.f : z;
  return from_float<T>(z);
}

// Each of a pair of floats as the sum of three bfloat16 numbers (the first one's in the low halves), each the next eight bits, cut and not rounded: the sum is
// x to the last bit, and none of them is an infinity that x is not.  NaN is its first part.  Where the second or third part would be zero it is the
// smallest number of x's sign, 2^-133, unless the first is zero: so all products of an infinity with the parts of a number are infinities of one
// sign, and with zero none is a number.
__device__ __forceinline__ void split3(float x, float y, uint32_t (&p)[3]) {
  float r[2] = {x, y};
  const bool finite[2] = {fabsf(x) <= 3.402823466e38f, fabsf(y) <= 3.402823466e38f};
#pragma unroll
  for (int i = 0; i < 3; i++) {
    uint32_t bits[2];
#pragma unroll
    for (int k = 0; k < 2; k++) {
      bits[k] = __float_as_uint(r[k]) & 0xffff0000u;
      if (i == 0 && r[k] != r[k]) bits[k] = 0x7fc00000u;
      r[k] = finite[k] ? r[k] - __uint_as_float(bits[k]) : 0.f;
    }
    p[i] = __byte_perm(bits[0], bits[1], 0x7632);
  }
  uint32_t least;   // of the two halves: 0 or 1, and the sign; a part has that sign or is zero, so the larger as a whole number is the part where there is one
  asm("min.u16x2 %0, %1, %2;" : "=r"(least) : "r"(p[0] & 0x7fff7fffu), "r"(0x00010001u));
  least |= p[0] & 0x80008000u;
#pragma unroll
  for (int i = 1; i < 3; i++) asm("max.u16x2 %0, %1, %2;" : "=r"(p[i]) : "r"(p[i]), "r"(least));
}
#endif

}  // namespace gelib_b200
