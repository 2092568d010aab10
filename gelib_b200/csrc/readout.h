// What the readout's kernels (group norm, dense layers) and the optimizer step share: element types, wide accesses, activations.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.h"
#ifdef __CUDACC__
#include "f32x2.h"
#endif

namespace gelib_b200 {

inline bool known_type(int type) { return type == GELIB_F32 || type == GELIB_BF16 || type == GELIB_F16; }
inline bool known_activation(int act) { return act >= GELIB_ACT_NONE && act <= GELIB_ACT_GELU_TANH; }
inline int type_bytes(int type) { return type == GELIB_F32 ? 4 : 2; }
inline bool is_aligned(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// What a launch just made comes to.
inline int launched(const char* fn) {
  count_launch();
  GELIB_CUDA_TRY(fn, cudaGetLastError());
  return GELIB_OK;
}

// gw[c] and gb[c] from `parts` rows of partial sums each, (2, parts, n) floats; either may be null.
int launch_sum_parts(void* gw, void* gb, const float* sums, int parts, int n, int type, cudaStream_t stream);

#ifdef __CUDACC__

// Kernels of one call that follow one another: the later one is launched while the earlier one ends, and its blocks wait where they begin to read (or
// write) what that one wrote.  Every block that does so waits, and at least one block in any case: a kernel has ended when all its blocks have, so nothing that
// comes after can then begin before the earlier kernel has ended.
__device__ __forceinline__ void let_next_begin() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void await_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <class... P, class... A>
int launch_after(const char* fn, bool follows, void (*kernel)(P...), dim3 grid, dim3 block, size_t shared, cudaStream_t stream, const A&... args) {
  cudaLaunchConfig_t c = {};
  c.gridDim = grid, c.blockDim = block, c.dynamicSmemBytes = shared, c.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  c.attrs = at;
  c.numAttrs = follows ? 1 : 0;
  GELIB_CUDA_TRY(fn, cudaLaunchKernelEx(&c, kernel, args...));
  return launched(fn);
}

template <class T>
__device__ __forceinline__ float to_float(T v) {
  if constexpr (std::is_same_v<T, float>) return v;
  else if constexpr (std::is_same_v<T, __nv_bfloat16>) return __bfloat162float(v);
  else return __half2float(v);
}
template <class T>
__device__ __forceinline__ T from_float(float v) {
  if constexpr (std::is_same_v<T, float>) return v;
  else if constexpr (std::is_same_v<T, __nv_bfloat16>) return __float2bfloat16_rn(v);
  else return __float2half_rn(v);
}

template <int kBytes>
struct Raw;
template <>
struct Raw<16> { using type = uint4; };
template <>
struct Raw<8> { using type = uint2; };
template <>
struct Raw<4> { using type = uint32_t; };
template <>
struct Raw<2> { using type = uint16_t; };

// Numbers as they lie, and in float; 16-bit ones in pairs, which is half the instructions.
template <class T, int V>
__device__ __forceinline__ void unpack(const typename Raw<V * sizeof(T)>::type& raw, float (&x)[V]) {
  if constexpr (sizeof(T) == 2 && V % 2 == 0) {
    union { typename Raw<V * sizeof(T)>::type raw; uint32_t u[V / 2]; } w;
    w.raw = raw;
#pragma unroll
    for (int k = 0; k < V / 2; k++) {
      if constexpr (std::is_same_v<T, __nv_bfloat16>) {
        x[2 * k] = __uint_as_float(w.u[k] << 16);
        x[2 * k + 1] = __uint_as_float(w.u[k] & 0xffff0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w.u[k]));
        x[2 * k] = f.x, x[2 * k + 1] = f.y;
      }
    }
  } else {
    union { typename Raw<V * sizeof(T)>::type raw; T t[V]; } w;
    w.raw = raw;
#pragma unroll
    for (int k = 0; k < V; k++) x[k] = to_float(w.t[k]);
  }
}
template <class T, int V>
__device__ __forceinline__ typename Raw<V * sizeof(T)>::type pack(const float (&x)[V]) {
  if constexpr (sizeof(T) == 2 && V % 2 == 0) {
    union { typename Raw<V * sizeof(T)>::type raw; uint32_t u[V / 2]; } w;
#pragma unroll
    for (int k = 0; k < V / 2; k++) {
      if constexpr (std::is_same_v<T, __nv_bfloat16>) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * k], x[2 * k + 1]);
        w.u[k] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __half2 h = __floats2half2_rn(x[2 * k], x[2 * k + 1]);
        w.u[k] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    return w.raw;
  } else {
    union { typename Raw<V * sizeof(T)>::type raw; T t[V]; } w;
#pragma unroll
    for (int k = 0; k < V; k++) w.t[k] = from_float<T>(x[k]);
    return w.raw;
  }
}

// V consecutive elements as one access of V * sizeof(T) bytes.
template <class T, int V>
__device__ __forceinline__ void load_vec(const T* src, float (&x)[V]) {
  unpack<T, V>(*reinterpret_cast<const typename Raw<V * sizeof(T)>::type*>(src), x);
}
template <class T, int V>
__device__ __forceinline__ void store_vec(T* dst, const float (&x)[V]) {
  *reinterpret_cast<typename Raw<V * sizeof(T)>::type*>(dst) = pack<T, V>(x);
}

// V numbers at a time, in packed pairs: half the instructions.  d may be any of the operands.
template <int V>
__device__ __forceinline__ void fma_all(float (&d)[V], const float (&a)[V], const float (&b)[V], const float (&c)[V]) {
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int k = 0; k < V; k += 2) unpack2(fma2(pack2(a[k], a[k + 1]), pack2(b[k], b[k + 1]), pack2(c[k], c[k + 1])), d[k], d[k + 1]);
  } else {
#pragma unroll
    for (int k = 0; k < V; k++) d[k] = fmaf(a[k], b[k], c[k]);
  }
}
template <int V>
__device__ __forceinline__ void fma_all(float (&d)[V], const float (&a)[V], float b, float c) {
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int k = 0; k < V; k += 2) unpack2(fma2(pack2(a[k], a[k + 1]), pack2(b, b), pack2(c, c)), d[k], d[k + 1]);
  } else {
#pragma unroll
    for (int k = 0; k < V; k++) d[k] = fmaf(a[k], b, c);
  }
}
template <int V>
__device__ __forceinline__ void fma_all(float (&d)[V], const float (&a)[V], float b, const float (&c)[V]) {
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int k = 0; k < V; k += 2) unpack2(fma2(pack2(a[k], a[k + 1]), pack2(b, b), pack2(c[k], c[k + 1])), d[k], d[k + 1]);
  } else {
#pragma unroll
    for (int k = 0; k < V; k++) d[k] = fmaf(a[k], b, c[k]);
  }
}
template <int V>
__device__ __forceinline__ void mul_all(float (&d)[V], const float (&a)[V], const float (&b)[V]) {
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int k = 0; k < V; k += 2) unpack2(mul2(pack2(a[k], a[k + 1]), pack2(b[k], b[k + 1])), d[k], d[k + 1]);
  } else {
#pragma unroll
    for (int k = 0; k < V; k++) d[k] = a[k] * b[k];
  }
}
template <int V>
__device__ __forceinline__ void mul_all(float (&d)[V], const float (&a)[V], float b) {
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int k = 0; k < V; k += 2) unpack2(mul2(pack2(a[k], a[k + 1]), pack2(b, b)), d[k], d[k + 1]);
  } else {
#pragma unroll
    for (int k = 0; k < V; k++) d[k] = a[k] * b;
  }
}
template <int V>
__device__ __forceinline__ void add_all(float (&d)[V], const float (&a)[V], const float (&b)[V]) {
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int k = 0; k < V; k += 2) unpack2(add2(pack2(a[k], a[k + 1]), pack2(b[k], b[k + 1])), d[k], d[k + 1]);
  } else {
#pragma unroll
    for (int k = 0; k < V; k++) d[k] = a[k] + b[k];
  }
}
template <int V>
__device__ __forceinline__ void add_all(float (&d)[V], const float (&a)[V], float b) {
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int k = 0; k < V; k += 2) unpack2(add2(pack2(a[k], a[k + 1]), pack2(b, b)), d[k], d[k + 1]);
  } else {
#pragma unroll
    for (int k = 0; k < V; k++) d[k] = a[k] + b;
  }
}
template <int V>
__device__ __forceinline__ float sum_of(const float (&a)[V]) {
  if constexpr (V % 2 == 0) {
    f32x2 s = pack2(a[0], a[1]);
#pragma unroll
    for (int k = 2; k < V; k += 2) s = add2(s, pack2(a[k], a[k + 1]));
    float x, y;
    unpack2(s, x, y);
    return x + y;
  } else {
    float s = a[0];
#pragma unroll
    for (int k = 1; k < V; k++) s += a[k];
    return s;
  }
}
template <int V>
__device__ __forceinline__ float dot_of(const float (&a)[V], const float (&b)[V]) {
  if constexpr (V % 2 == 0) {
    f32x2 s = mul2(pack2(a[0], a[1]), pack2(b[0], b[1]));
#pragma unroll
    for (int k = 2; k < V; k += 2) s = fma2(pack2(a[k], a[k + 1]), pack2(b[k], b[k + 1]), s);
    float x, y;
    unpack2(s, x, y);
    return x + y;
  } else {
    float s = a[0] * b[0];
#pragma unroll
    for (int k = 1; k < V; k++) s = fmaf(a[k], b[k], s);
    return s;
  }
}

// q = 1 / (1 + 2^t), from the approximations of 2^x and 1 / x without their treatment of subnormal numbers, which took most of the instructions: where
// 2^t is subnormal it is nothing beside 1, and where 1 + 2^t is so large that the quotient is subnormal, that is 0 here.
template <int V>
__device__ __forceinline__ void logistics(float (&q)[V], const float (&t)[V]) {
#pragma unroll
  for (int k = 0; k < V; k++) asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(q[k]) : "f"(t[k]));
  add_all(q, q, 1.f);
#pragma unroll
  for (int k = 0; k < V; k++) asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(q[k]) : "f"(q[k]));
}
constexpr float kLog2e = 1.4426950408889634f;

constexpr float kGelu0 = 1.5957691216057308f;             // 2 sqrt(2 / pi): 0.5 (1 + tanh u) is the logistic function of 2u
constexpr float kGelu1 = kGelu0 * 0.044715f;

// x = act(x)
template <int V>
__device__ __forceinline__ void activate(float (&x)[V], int act) {
  if (act == GELIB_ACT_NONE) return;
  if (act == GELIB_ACT_RELU) {
#pragma unroll
    for (int k = 0; k < V; k++) x[k] = x[k] < 0.f ? 0.f : x[k];     // NaN stays NaN
    return;
  }
  float t[V];
  if (act == GELIB_ACT_SILU) {
    mul_all(t, x, -kLog2e);
  } else {
    mul_all(t, x, x);
    fma_all(t, t, -kLog2e * kGelu1, -kLog2e * kGelu0);
    mul_all(t, t, x);
  }
  logistics(t, t);
  mul_all(x, x, t);
}

// g = g act'(z)
template <int V>
__device__ __forceinline__ void activate_back(float (&g)[V], const float (&z)[V], int act) {
  if (act == GELIB_ACT_NONE) return;
  if (act == GELIB_ACT_RELU) {
#pragma unroll
    for (int k = 0; k < V; k++) g[k] = z[k] > 0.f ? g[k] : z[k] != z[k] ? z[k] : 0.f;
    return;
  }
  float q[V], u[V];
  if (act == GELIB_ACT_SILU) {   // q + z q (1 - q)
    mul_all(q, z, -kLog2e);
    logistics(q, q);
    fma_all(u, q, -1.f, 1.f);
    mul_all(u, u, z);
    fma_all(q, q, u, q);
  } else {                       // q + q (1 - q) z (k0 + 3 k1 z^2)
    float z2[V];
#pragma unroll
    for (int k = 0; k < V; k++) z2[k] = fminf(z[k] * z[k], 1e30f);
    fma_all(q, z2, -kLog2e * kGelu1, -kLog2e * kGelu0);
    mul_all(q, q, z);
    logistics(q, q);
    // q (1 - q) first: beyond |z| = 12 it is 0, and 0 times a finite z and the finite third factor stays 0; those two together may be an infinity
    fma_all(u, q, -1.f, 1.f);
    mul_all(u, u, q);
    mul_all(u, u, z);
    fma_all(z2, z2, 3.f * kGelu1, kGelu0);
    fma_all(q, u, z2, q);
  }
  mul_all(g, g, q);
}

#endif

}  // namespace gelib_b200
