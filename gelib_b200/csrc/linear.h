// Dense layers: what the C ABI hands to the kernels, and the matrix product that they are made of.
#pragma once
#include "common.h"

namespace gelib_b200 {

// One operand of D = A B: element (i, k) at base[i * si + k * sk]; one of the strides is 1 (i: the row of A, the column of B).
struct Operand {
  const void* base;
  long long si, sk;
};

// What happens to a sum d before it is stored: z = d + bias, y = act(z) + residual; z is stored too where it is asked for.
struct Epilogue {
  void* y;
  void* z;                 // or null
  const void *bias, *residual;   // or null
  int act;
};

struct Gemm {
  Operand a, b;
  Epilogue e;
  long long M, N, K;
  int type;
};

long long linear_workspace(const gelib_linear_args& p, bool backward);
int launch_linear(const gelib_linear_args& p, void* workspace, cudaStream_t stream);
int launch_linear_back(const gelib_linear_args& p, void* workspace, cudaStream_t stream);

}  // namespace gelib_b200
