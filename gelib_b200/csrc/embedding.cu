// Rows of a table by their numbers, and the gradient of the table:
//
//   y[i] = scale w[ids[i]],   gw[r] = scale sum of gy[i] over the i with ids[i] = r
//
// Both are bound by memory: forward reads the rows that are met and writes y, backward reads gy and writes all of gw.
#include <algorithm>
#include <cmath>

#include "heads.h"

namespace gelib_b200 {

namespace {

constexpr int kThreads = 256;

template <class T, int V>
__global__ void __launch_bounds__(kThreads) embedding_kernel(const EmbeddingCall c) {
  const int chunks = c.d / V;
  const long long all = c.n * chunks;
  for (long long e = (long long)blockIdx.x * kThreads + threadIdx.x; e < all; e += (long long)gridDim.x * kThreads) {
    const long long i = e / chunks, col = (e - i * chunks) * V, id = index_at(c.ids, i, c.index_bytes);
    float x[V];
    if (id >= 0 && id < c.v) {
      load_vec<T, V>(static_cast<const T*>(c.weight) + id * c.ldw + col, x);
      mul_all(x, x, c.scale);
    } else {
#pragma unroll
      for (int k = 0; k < V; k++) x[k] = NAN;
    }
    store_vec<T, V>(static_cast<T*>(c.y) + i * c.d + col, x);
  }
}

// A warp owns a row of the table and 32 V of its columns, and looks through all numbers for its own.
template <class T, int V>
__global__ void __launch_bounds__(kThreads) embedding_back_kernel(const EmbeddingCall c) {
  const int lane = threadIdx.x % 32, slabs = (c.d + 32 * V - 1) / (32 * V);
  const long long at = (long long)blockIdx.x * (kThreads / 32) + threadIdx.x / 32, row = at / slabs;
  const int col = ((int)(at - row * slabs) * 32 + lane) * V;
  if (row >= c.v) return;
  float s[V];
#pragma unroll
  for (int k = 0; k < V; k++) s[k] = 0;
  if (row != c.padding)
    for (long long i0 = 0; i0 < c.n; i0 += 32) {
      unsigned found = __ballot_sync(0xffffffffu, i0 + lane < c.n && index_at(c.ids, i0 + lane, c.index_bytes) == row);
      while (found) {
        const long long i = i0 + __ffs(found) - 1;
        found &= found - 1;
        if (col < c.d) {
          float g[V];
          load_vec<T, V>(static_cast<const T*>(c.gy) + i * c.d + col, g);
          add_all(s, s, g);
        }
      }
    }
  if (col >= c.d) return;
  mul_all(s, s, c.scale);
  store_vec<T, V>(static_cast<T*>(c.gw) + row * c.d + col, s);
}

template <class T>
int launch_forward_as(const EmbeddingCall& c, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  const bool wide = c.d % V == 0 && c.ldw % V == 0 && is_aligned(c.y, 16) && is_aligned(c.weight, 16);
  const long long chunks = c.n * (wide ? c.d / V : c.d);
  const unsigned blocks = (unsigned)std::min((chunks + kThreads - 1) / kThreads, 148LL * 64);
  if (wide) embedding_kernel<T, V><<<blocks, kThreads, 0, stream>>>(c);
  else embedding_kernel<T, 1><<<blocks, kThreads, 0, stream>>>(c);
  return launched("embedding");
}

template <class T>
int launch_backward_as(const EmbeddingCall& c, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  const bool wide = c.d % V == 0 && is_aligned(c.gw, 16) && is_aligned(c.gy, 16);
  const long long columns = 32 * (wide ? V : 1), warps = (long long)c.v * ((c.d + columns - 1) / columns), blocks = (warps + kThreads / 32 - 1) / (kThreads / 32);
  if (blocks > 0x7fffffffLL) return fail(GELIB_INVALID, "embedding_back", "too many elements");
  if (wide) embedding_back_kernel<T, V><<<(unsigned)blocks, kThreads, 0, stream>>>(c);
  else embedding_back_kernel<T, 1><<<(unsigned)blocks, kThreads, 0, stream>>>(c);
  return launched("embedding_back");
}

}  // namespace

long long embedding_workspace(long long, int, int, int) { return 0; }

int launch_embedding(const EmbeddingCall& c, cudaStream_t stream) {
  return c.type == GELIB_F32 ? launch_forward_as<float>(c, stream) : c.type == GELIB_BF16 ? launch_forward_as<__nv_bfloat16>(c, stream) : launch_forward_as<__half>(c, stream);
}

int launch_embedding_back(const EmbeddingCall& c, void*, cudaStream_t stream) {
  return c.type == GELIB_F32 ? launch_backward_as<float>(c, stream) : c.type == GELIB_BF16 ? launch_backward_as<__nv_bfloat16>(c, stream) : launch_backward_as<__half>(c, stream);
}

}  // namespace gelib_b200
