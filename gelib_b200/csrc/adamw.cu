// AdamW over many tensors in one launch:
//
//   m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g^2,
//   p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// in 32 bits.  A 16-bit parameter has a 32-bit master copy that takes the step, and is the copy rounded; complex parameters are
// pairs of real ones.  The moments are held in 32 bits, or in 8: blocks of 256 elements share a power of two, codes are e4m3, and of v
// the root is held, whose range is half of v's in powers of two.  A moment that changes by a thousandth of itself a step would never leave its
// code if it were rounded to nearest, so rounding is stochastic, from a hash of the call's seed and the element's number; the root is
// never rounded to zero while v is above it, which would divide by eps.  Where the caller asks for it a master copy whose rounding is not the parameter
// becomes the parameter first, which is two bytes more to read.
//
// The step is bound by memory: 28 bytes an element in 32 bits (p, m, v read and written, g read), 16 in 8 bits.  A network's weights
// are many small tensors, so their addresses travel in the launch's parameters, a tensor is cut into pieces of as many elements as a block takes, and
// a block finds its piece by bisection.
//
// Measured on 46.7 million weights: 190 us in 32 bits (28 bytes an element, 6.8 TB/s: the copy rate); 8 bits and a bfloat16 head 222 us with the values of both
// moments written out (two launches of 27), where the step's bytes take 114.  Its 85 instructions an element, most of them the two roundings, fill 65 % of the issue
// slots and 56 % of the integer pipe, DRAM is at 48 %: loads and arithmetic of a piece follow one another, and 36 warps of an SM do not cover
// that.  Two dozen small tensors 11 us a call, half of it Python's.
#include <cuda_fp8.h>

#include <algorithm>
#include <cmath>

#include "readout.h"

namespace gelib_b200 {

namespace {

constexpr int kThreads = 256;
constexpr int kBlock = 256;        // elements that share a scale
constexpr int kPiece = 2048;       // elements of a block of threads

struct Entry {
  void* p;           // the parameter: float, or 16 bits wide beside `master`
  float* master;     // null for a float parameter
  const void* g;     // in the parameter's type
  void *m, *v;       // float, or codes
  float *ms, *vs;    // scales of the codes
  long long n;
  int first;         // number of the tensor's first piece in this launch
  int kind;          // type of p and g; bit 8: all pointers allow wide accesses
  long long at;      // number of its first block of 256 elements in the call: the hash counts elements of padded tensors
};

struct Scalars {
  float b1, one_b1, b2, one_b2, keep, step, root, eps;   // keep = 1 - lr wd, step = lr / (1 - b1^t), root = 1 / sqrt(1 - b2^t)
  const float* grad_scale;
  unsigned seed_mix;
  int refresh;
};

template <int N>
struct Args {
  Scalars s;
  int count;
  Entry e[N];
};

// Two rounds of multiplication and shifts; h is the element's number and the seed, each times an odd number.
__device__ __forceinline__ unsigned random_bits(unsigned h) {
  h = (h ^ (h >> 15)) * 0x2C1B3C6Du;
  h = (h ^ (h >> 12)) * 0x297A2D39u;
  return h ^ (h >> 15);
}

// Eight elements.  The approximate reciprocal, and the approximate root where it is not kept, are a unit or two in the last place off, which the step may be too.
//
// kRoot: r becomes the new root of v, to be rounded to a code.  There a last place matters: where it moves a value over the point at which the
// hash takes the other neighbour, the code is an eighth off.  So each product and sum is rounded by itself, in the formula's order (a packed product and
// a packed sum were joined by the compiler: 8 codes of 2^24 differed), and the root is the one rounded to nearest.
template <bool kRoot>
__device__ __forceinline__ void update(const Scalars& s, float (&g)[8], float (&p)[8], float (&m)[8], float (&v)[8], float (&r)[8]) {
  float t[8];
  mul_all(m, m, s.b1);
  mul_all(v, v, s.b2);
  if constexpr (kRoot) {
    float h[8];
    mul_all(h, g, s.one_b1);
    mul_all(t, g, s.one_b2);
    mul_all(t, t, g);
#pragma unroll
    for (int k = 0; k < 8; k++) {
      m[k] = __fadd_rn(m[k], h[k]);
      v[k] = __fadd_rn(v[k], t[k]);
    }
  } else {
    fma_all(m, g, s.one_b1, m);
    mul_all(t, g, g);
    fma_all(v, t, s.one_b2, v);
  }
#pragma unroll
  for (int k = 0; k < 8; k++) {
    if constexpr (kRoot) r[k] = __fsqrt_rn(v[k]);
    else asm("sqrt.approx.f32 %0, %1;" : "=f"(r[k]) : "f"(v[k]));
  }
  fma_all(t, r, s.root, s.eps);
#pragma unroll
  for (int k = 0; k < 8; k++) asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t[k]) : "f"(t[k]));
  mul_all(t, t, m);
  mul_all(p, p, s.keep);
  fma_all(p, t, -s.step, p);
}

// The power of two that brings `top` into [128, 256): codes then reach 256 after rounding up, below e4m3's 448.  No smaller than
// 2^-100, so that scale times code stays a normal number; a block whose values are all zero has that scale too.
__device__ __forceinline__ int scale_exponent(float top) { return max((int)(__float_as_uint(top) >> 23) - 127 - 7, -100); }

// 0 <= y < 256 on the grid of e4m3: three bits of mantissa, steps of 2^-9 below 2^-6; u in [0, 2^16), sixteen times it and 8 more, decides between the
// neighbours.  What is no finite number becomes NaN.
__device__ __forceinline__ float on_grid(float y, unsigned u16) {
  const float more = y < 0.015625f ? 0.015625f : 0.f;
  const float q = __uint_as_float((__float_as_uint(y + more) + u16) & 0xfff00000u);
  return fmaf(y, 0.f, q - more);
}

// Pairs of codes and their values, the first in the low byte.
__device__ __forceinline__ unsigned short codes_of(float q0, float q1) { return __nv_cvt_float2_to_fp8x2(make_float2(q0, q1), __NV_SATFINITE, __NV_E4M3); }
__device__ __forceinline__ float2 values_of(unsigned short c) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(c, __NV_E4M3);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

template <int N>
__device__ __forceinline__ const Entry& find(const Args<N>& a, int piece) {
  int lo = 0, hi = a.count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.e[mid].first <= piece) lo = mid; else hi = mid;
  }
  return a.e[lo];
}

template <class T, bool kWide>
__device__ __forceinline__ void load_n(const T* src, long long i, long long n, float (&x)[8]) {
  if constexpr (kWide) {
    if (i + 8 <= n) {
      if constexpr (sizeof(T) == 4) {
        const float4 a = *reinterpret_cast<const float4*>(src + i), b = *reinterpret_cast<const float4*>(src + i + 4);
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
      } else {
        load_vec<T, 8>(src + i, x);
      }
      return;
    }
  }
#pragma unroll
  for (int k = 0; k < 8; k++) x[k] = i + k < n ? to_float(src[i + k]) : 0.f;
}

template <class T, bool kWide>
__device__ __forceinline__ void store_n(T* dst, long long i, long long n, const float (&x)[8]) {
  if constexpr (kWide) {
    if (i + 8 <= n) {
      if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(dst + i) = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4*>(dst + i + 4) = make_float4(x[4], x[5], x[6], x[7]);
      } else {
        store_vec<T, 8>(dst + i, x);
      }
      return;
    }
  }
#pragma unroll
  for (int k = 0; k < 8; k++)
    if (i + k < n) dst[i + k] = from_float<T>(x[k]);
}

template <bool kWide>
__device__ __forceinline__ void load_codes(const unsigned char* src, long long i, long long n, unsigned short (&c)[4]) {
  union { uint2 u; unsigned short p[4]; unsigned char c[8]; } w;
  if (kWide && i + 8 <= n) {
    w.u = *reinterpret_cast<const uint2*>(src + i);
  } else {
#pragma unroll
    for (int k = 0; k < 8; k++) w.c[k] = i + k < n ? src[i + k] : 0;
  }
#pragma unroll
  for (int k = 0; k < 4; k++) c[k] = w.p[k];
}

template <bool kWide>
__device__ __forceinline__ void store_codes(unsigned char* dst, long long i, long long n, const unsigned short (&c)[4]) {
  union { uint2 u; unsigned short p[4]; unsigned char c[8]; } w;
#pragma unroll
  for (int k = 0; k < 4; k++) w.p[k] = c[k];
  if (kWide && i + 8 <= n) {
    *reinterpret_cast<uint2*>(dst + i) = w.u;
    return;
  }
#pragma unroll
  for (int k = 0; k < 8; k++)
    if (i + k < n) dst[i + k] = w.c[k];
}

// A lane's eight consecutive elements; with 8-bit states a warp's 256 are one block.
template <class T, bool k8, bool kWide>
__device__ __forceinline__ void step_piece(const Entry& e, const Scalars& s, long long i) {
  const long long n = e.n;
  if ((i & ~(long long)(kBlock - 1)) >= n) return;   // the whole warp
  float p[8], g[8], m[8], v[8];
  float* master = sizeof(T) == 4 ? static_cast<float*>(e.p) : e.master;
  load_n<float, kWide>(master, i, n, p);
  load_n<T, kWide>(static_cast<const T*>(e.g), i, n, g);
  if constexpr (sizeof(T) == 2) {
    if (s.refresh) {   // what was written to a parameter since the last step is not its master copy's rounding
      float q[8], held[8];
      load_n<T, kWide>(static_cast<const T*>(e.p), i, n, q);
      unpack<T, 8>(pack<T, 8>(p), held);
#pragma unroll
      for (int k = 0; k < 8; k++)
        if (__float_as_uint(held[k]) != __float_as_uint(q[k])) p[k] = q[k];
    }
  }
  unsigned char *mc = static_cast<unsigned char*>(e.m), *vc = static_cast<unsigned char*>(e.v);
  const long long block = i / kBlock;
  if constexpr (k8) {
    unsigned short a[4], b[4];
    load_codes<kWide>(mc, i, n, a);
    load_codes<kWide>(vc, i, n, b);
    const float ms = e.ms[block], vs = e.vs[block];
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const float2 p = values_of(a[k]), r = values_of(b[k]);
      m[2 * k] = p.x, m[2 * k + 1] = p.y, v[2 * k] = r.x, v[2 * k + 1] = r.y;
    }
    mul_all(m, m, ms);
    mul_all(v, v, vs);
    mul_all(v, v, v);
  } else {
    load_n<float, kWide>(static_cast<const float*>(e.m), i, n, m);
    load_n<float, kWide>(static_cast<const float*>(e.v), i, n, v);
  }
  if (s.grad_scale) mul_all(g, g, *s.grad_scale);
  float r[8];
  update<k8>(s, g, p, m, v, r);
  store_n<float, kWide>(master, i, n, p);
  if constexpr (sizeof(T) == 2) store_n<T, kWide>(static_cast<T*>(e.p), i, n, p);
  if constexpr (!k8) {
    store_n<float, kWide>(static_cast<float*>(e.m), i, n, m);
    store_n<float, kWide>(static_cast<float*>(e.v), i, n, v);
  } else {
    // a value that is no finite number spoils its own element and not its block: it takes no part in the scale
    constexpr float kMost = 3.402823466e38f;
    float tm = 0, tr = 0;
#pragma unroll
    for (int k = 0; k < 8; k++) tm = fmaxf(tm, fabsf(m[k])), tr = fmaxf(tr, r[k]);   // NaN drops out
    if (!(tm <= kMost && tr <= kMost)) {
      tm = tr = 0;
#pragma unroll
      for (int k = 0; k < 8; k++) {
        if (fabsf(m[k]) <= kMost) tm = fmaxf(tm, fabsf(m[k]));
        if (r[k] <= kMost) tr = fmaxf(tr, r[k]);
      }
    }
    // neither is negative: their order is that of their bits, and a warp has the largest of those in one step
    tm = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(tm)));
    tr = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(tr)));
    const int em = scale_exponent(tm), er = scale_exponent(tr);
    const float im = __uint_as_float((127 - em) << 23), ir = __uint_as_float((127 - er) << 23);
    const unsigned long long number = (unsigned long long)e.at * kBlock + (unsigned long long)i;
    unsigned h = (unsigned)number * 0x9E3779B1u + (unsigned)(number >> 32) * 0x7FEB352Du + s.seed_mix;   // eight elements lie in one multiple of 2^32
    unsigned short a[4], b[4];
#pragma unroll
    for (int k = 0; k < 8; k += 2) {
      float qm[2], qr[2];
#pragma unroll
      for (int j = 0; j < 2; j++) {
        const unsigned u = random_bits(h);
        h += 0x9E3779B1u;
        qm[j] = copysignf(on_grid(fabsf(m[k + j]) * im, (u & 0xffff) * 16 + 8), m[k + j]);
        qr[j] = on_grid(r[k + j] * ir, (u >> 12 & 0xffff0) + 8);
        if (r[k + j] > 0 && qr[j] < 0.001953125f) qr[j] = 0.001953125f;
      }
      a[k / 2] = codes_of(qm[0], qm[1]);
      b[k / 2] = codes_of(qr[0], qr[1]);
    }
    store_codes<kWide>(mc, i, n, a);
    store_codes<kWide>(vc, i, n, b);
    if ((threadIdx.x & 31) == 0) {
      e.ms[block] = __uint_as_float((em + 127) << 23);
      e.vs[block] = __uint_as_float((er + 127) << 23);
    }
  }
}

// Five blocks of an SM although registers spill: a pass over 46.7 million weights, with the values of both moments, 222 us in 8 bits; six took 4 us more.
template <int N, bool k8>
__global__ void __launch_bounds__(kThreads, k8 ? 5 : 4) adamw_kernel(const __grid_constant__ Args<N> a) {
  const Entry& e = find(a, (int)blockIdx.x);
  const long long i = (long long)((int)blockIdx.x - e.first) * kPiece + threadIdx.x * 8;
  static_assert(kPiece == kThreads * 8, "a lane takes eight elements");
  const bool wide = e.kind & 8;
  switch (e.kind & 7) {
    case GELIB_F32:
      wide ? step_piece<float, k8, true>(e, a.s, i) : step_piece<float, k8, false>(e, a.s, i);
      break;
    case GELIB_BF16:
      wide ? step_piece<__nv_bfloat16, k8, true>(e, a.s, i) : step_piece<__nv_bfloat16, k8, false>(e, a.s, i);
      break;
    default:
      wide ? step_piece<__half, k8, true>(e, a.s, i) : step_piece<__half, k8, false>(e, a.s, i);
  }
}

template <int N, bool k8>
int launch(const gelib_adamw_tensor* t, const long long* first_block, int count, const Scalars& s, int pieces, cudaStream_t stream) {
  static thread_local Args<N> a;
  a.s = s;
  a.count = count;
  int first = 0;
  for (int i = 0; i < count; i++) {
    const gelib_adamw_tensor& x = t[i];
    const int state = k8 ? 8 : 16;
    const bool wide = is_aligned(x.p, 16) && is_aligned(x.g, 16) && is_aligned(x.master, 16) && is_aligned(x.m, state) && is_aligned(x.v, state);
    a.e[i] = {x.p, x.master, x.g, x.m, x.v, x.m_scale, x.v_scale, x.n, first, x.type | (wide ? 8 : 0), first_block[i]};
    first += (int)((x.n + kPiece - 1) / kPiece);
  }
  adamw_kernel<N, k8><<<pieces, kThreads, 0, stream>>>(a);
  return launched("adamw_step");
}

constexpr int kMost = 350;   // entries of 80 bytes
static_assert(sizeof(Args<kMost>) <= 32764, "what a launch's parameters may have");

__global__ void __launch_bounds__(kThreads) block8_values_kernel(__nv_bfloat16* __restrict__ out, const unsigned char* __restrict__ codes,
                                                                const float* __restrict__ scale, long long n, bool wide) {
  // two accesses a thread, asked for together
  const long long i0 = ((long long)blockIdx.x * 2 * kThreads + threadIdx.x) * 8;
  unsigned short c[2][4];
  float s[2];
#pragma unroll
  for (int q = 0; q < 2; q++) {
    const long long i = i0 + q * kThreads * 8;
    if (i < n) {
      wide ? load_codes<true>(codes, i, n, c[q]) : load_codes<false>(codes, i, n, c[q]);
      s[q] = scale[i / kBlock];
    }
  }
#pragma unroll
  for (int q = 0; q < 2; q++) {
    const long long i = i0 + q * kThreads * 8;
    if (i >= n) return;
    float x[8];
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const float2 f = values_of(c[q][k]);
      x[2 * k] = f.x, x[2 * k + 1] = f.y;
    }
    mul_all(x, x, s[q]);
    wide ? store_n<__nv_bfloat16, true>(out, i, n, x) : store_n<__nv_bfloat16, false>(out, i, n, x);
  }
}

}  // namespace

int launch_adamw(int count, const gelib_adamw_tensor* t, const gelib_adamw_options& o, cudaStream_t stream) {
  Scalars s;
  const double c1 = 1 - std::pow(o.beta1, (double)o.step), c2 = 1 - std::pow(o.beta2, (double)o.step);
  s.b1 = (float)o.beta1, s.one_b1 = (float)(1 - o.beta1), s.b2 = (float)o.beta2, s.one_b2 = (float)(1 - o.beta2);
  s.keep = (float)(1 - o.lr * o.weight_decay), s.step = (float)(o.lr / c1), s.root = (float)(1 / std::sqrt(c2)), s.eps = (float)o.eps;
  s.grad_scale = o.grad_scale, s.refresh = o.refresh_master;
  s.seed_mix = (unsigned)o.seed * 0x6A09E667u + (unsigned)(o.seed >> 32) * 0x3C6EF373u;
  const bool k8 = o.state_bits == 8;
  std::vector<gelib_adamw_tensor> group;
  std::vector<long long> blocks;
  long long block = 0, pieces = 0;
  auto flush = [&]() -> int {
    const int n = (int)group.size();
    if (n == 0) return GELIB_OK;
    const int p = (int)pieces;
    int st;
    // the parameters of a launch are copied whatever the number of tensors: few of them take a small set
    if (n <= 32) st = k8 ? launch<32, true>(group.data(), blocks.data(), n, s, p, stream) : launch<32, false>(group.data(), blocks.data(), n, s, p, stream);
    else st = k8 ? launch<kMost, true>(group.data(), blocks.data(), n, s, p, stream) : launch<kMost, false>(group.data(), blocks.data(), n, s, p, stream);
    group.clear();
    blocks.clear();
    pieces = 0;
    return st;
  };
  for (int i = 0; i < count; i++) {
    // a tensor of more pieces than a launch counts goes in parts; their length is a multiple of a block of 256
    const long long most = (long long)kPiece << 29;
    for (long long at = 0; at < t[i].n; at += most) {
      gelib_adamw_tensor x = t[i];
      const long long width = type_bytes(x.type), state = k8 ? 1 : 4;
      x.p = (char*)x.p + at * width, x.g = (const char*)x.g + at * width;
      if (x.master) x.master += at;
      x.m = (char*)x.m + at * state, x.v = (char*)x.v + at * state;
      if (k8) x.m_scale += at / kBlock, x.v_scale += at / kBlock;
      x.n = std::min(most, t[i].n - at);
      const long long need = (x.n + kPiece - 1) / kPiece;
      if ((int)group.size() == kMost || pieces + need > 0x7fffffffLL) {
        const int st = flush();
        if (st != GELIB_OK) return st;
      }
      group.push_back(x);
      blocks.push_back(block + at / kBlock);
      pieces += need;
    }
    block += (t[i].n + kBlock - 1) / kBlock;
  }
  return flush();
}

int launch_block8_values(void* out, const void* codes, const float* scale, long long n, cudaStream_t stream) {
  if (n == 0) return GELIB_OK;
  const bool wide = is_aligned(out, 16) && is_aligned(codes, 8);
  const long long per = kThreads * 16, blocks = (n + per - 1) / per;
  if (blocks > 0x7fffffffLL) return fail(GELIB_INVALID, "block8_values", "too many elements");
  block8_values_kernel<<<(unsigned)blocks, kThreads, 0, stream>>>((__nv_bfloat16*)out, (const unsigned char*)codes, scale, n, wide);
  return launched("block8_values");
}

}  // namespace gelib_b200
