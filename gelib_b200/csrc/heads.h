// Embedding tables and the losses behind a last dense layer: what the C ABI hands to the kernels.
#pragma once
#include "common.h"
#include "readout.h"

namespace gelib_b200 {

struct EmbeddingCall {
  void* y;               // forward: (n, d)
  void* gw;              // backward: (v, d)
  const void *ids, *weight, *gy;
  long long n, ldw, padding;
  int v, d, index_bytes, type;
  float scale;
};
long long embedding_state_bytes(long long n, int v);
long long embedding_workspace(long long n, int v, int d, int type);
int launch_embedding(const EmbeddingCall& c, void* state, cudaStream_t stream);
int launch_embedding_back(const EmbeddingCall& c, const void* state, void* workspace, cudaStream_t stream);

long long linear_loss_state_bytes(const gelib_linear_loss_args& p);
long long linear_loss_workspace(const gelib_linear_loss_args& p, bool backward);
int launch_linear_loss(const gelib_linear_loss_args& p, void* workspace, cudaStream_t stream);
int launch_linear_loss_back(const gelib_linear_loss_args& p, void* workspace, cudaStream_t stream);

#ifdef __CUDACC__
__device__ __forceinline__ long long index_at(const void* p, long long i, int bytes) {
  return bytes == 8 ? static_cast<const long long*>(p)[i] : static_cast<const int*>(p)[i];
}
#endif

}  // namespace gelib_b200
