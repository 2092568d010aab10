// Group norm: what the C ABI hands to the kernels.
#pragma once
#include "common.h"

namespace gelib_b200 {

struct GroupNormCall {
  void* y;                          // forward: y; backward: gx (may be null)
  float *mean, *rstd;               // (b, groups): written by the forward (may be null), read by the backward
  const void *x, *w, *bias, *gy;    // w, bias may be null; gy: null in the forward
  void *gw, *gb;                    // backward, may be null
  long long b, s;
  int n, groups;
  float eps;
  int act, type;
  float* workspace;
};

long long group_norm_workspace(long long b, long long s, int n, int groups, int type, bool backward);
int launch_group_norm(const GroupNormCall& c, cudaStream_t stream);

}  // namespace gelib_b200
