// AdamW over many tensors in one launch:
//
//   m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g^2,
//   p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// in 32 bits.  A 16-bit parameter has a 32-bit master copy that takes the step, and is the copy rounded; complex parameters are
// pairs of real ones.  The moments are held in 32 bits, or in 8: blocks of 256 elements share a power of two, codes are e4m3, and of v
// the root is held, whose range is half of v's in powers of two.  A moment that changes by a thousandth of itself a step would never leave its
// code if it were rounded to nearest, so rounding is stochastic, from a hash of the call's seed and the element's number; the root is
// never rounded to zero while v is above it, which would divide by eps.
//
// The step is bound by memory: 28 bytes an element in 32 bits (p, m, v read and written, g read), 16 in 8 bits.  A network's weights
// are many small tensors, so their addresses travel in the launch's parameters, a tensor is cut into pieces of as many elements as a block takes, and
// a block finds its piece by bisection.
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
};

template <int N>
struct Args {
  Scalars s;
  int count;
  Entry e[N];
};

// Two rounds of multiplication and shifts over the element's number and the seed.
__device__ __forceinline__ unsigned random_bits(unsigned seed_mix, unsigned long long i) {
  unsigned h = (unsigned)i * 0x9E3779B1u + (unsigned)(i >> 32) * 0x7FEB352Du + seed_mix;
  h = (h ^ (h >> 15)) * 0x2C1B3C6Du;
  h = (h ^ (h >> 12)) * 0x297A2D39u;
  return h ^ (h >> 15);
}

__device__ __forceinline__ void update(const Scalars& s, float g, float& p, float& m, float& v) {
  m = s.b1 * m + s.one_b1 * g;
  v = s.b2 * v + s.one_b2 * g * g;
  p = p * s.keep - s.step * m / (sqrtf(v) * s.root + s.eps);
}

// The power of two that brings `top` into [128, 256): codes then reach 256 after rounding up, below e4m3's 448.  No smaller than
// 2^-100, so that scale times code stays a normal number; a block whose values are all zero has that scale too.
__device__ __forceinline__ int scale_exponent(float top) { return max((int)(__float_as_uint(top) >> 23) - 127 - 7, -100); }

// |y| < 256 on the grid of e4m3: three bits of mantissa, steps of 2^-9 below 2^-6; u in [0, 2^16) decides between the neighbours.
__device__ __forceinline__ float on_grid(float y, unsigned u) {
  const bool small = y < 0.015625f;
  const float t = small ? y + 0.015625f : y;
  const float q = __uint_as_float((__float_as_uint(t) + (u * 16 + 8)) & 0xfff00000u);
  return small ? q - 0.015625f : q;
}

__device__ __forceinline__ unsigned char code_of(float q) { return (unsigned char)__nv_cvt_float_to_fp8(q, __NV_SATFINITE, __NV_E4M3); }
__device__ __forceinline__ float value_of(unsigned char c) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3)));
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
        union { uint4 u; T t[8]; } w;
        w.u = *reinterpret_cast<const uint4*>(src + i);
#pragma unroll
        for (int k = 0; k < 8; k++) x[k] = to_float(w.t[k]);
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
        union { uint4 u; T t[8]; } w;
#pragma unroll
        for (int k = 0; k < 8; k++) w.t[k] = from_float<T>(x[k]);
        *reinterpret_cast<uint4*>(dst + i) = w.u;
      }
      return;
    }
  }
#pragma unroll
  for (int k = 0; k < 8; k++)
    if (i + k < n) dst[i + k] = from_float<T>(x[k]);
}

template <bool kWide>
__device__ __forceinline__ void load_codes(const unsigned char* src, long long i, long long n, unsigned char (&c)[8]) {
  if (kWide && i + 8 <= n) {
    union { uint2 u; unsigned char c[8]; } w;
    w.u = *reinterpret_cast<const uint2*>(src + i);
#pragma unroll
    for (int k = 0; k < 8; k++) c[k] = w.c[k];
    return;
  }
#pragma unroll
  for (int k = 0; k < 8; k++) c[k] = i + k < n ? src[i + k] : 0;
}

template <bool kWide>
__device__ __forceinline__ void store_codes(unsigned char* dst, long long i, long long n, const unsigned char (&c)[8]) {
  if (kWide && i + 8 <= n) {
    union { uint2 u; unsigned char c[8]; } w;
#pragma unroll
    for (int k = 0; k < 8; k++) w.c[k] = c[k];
    *reinterpret_cast<uint2*>(dst + i) = w.u;
    return;
  }
#pragma unroll
  for (int k = 0; k < 8; k++)
    if (i + k < n) dst[i + k] = c[k];
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
  unsigned char *mc = static_cast<unsigned char*>(e.m), *vc = static_cast<unsigned char*>(e.v);
  const long long block = i / kBlock;
  if constexpr (k8) {
    unsigned char a[8], b[8];
    load_codes<kWide>(mc, i, n, a);
    load_codes<kWide>(vc, i, n, b);
    const float ms = e.ms[block], vs = e.vs[block];
#pragma unroll
    for (int k = 0; k < 8; k++) {
      m[k] = value_of(a[k]) * ms;
      const float r = value_of(b[k]) * vs;
      v[k] = r * r;
    }
  } else {
    load_n<float, kWide>(static_cast<const float*>(e.m), i, n, m);
    load_n<float, kWide>(static_cast<const float*>(e.v), i, n, v);
  }
  const float scale = s.grad_scale ? *s.grad_scale : 1.f;
#pragma unroll
  for (int k = 0; k < 8; k++) update(s, s.grad_scale ? g[k] * scale : g[k], p[k], m[k], v[k]);
  store_n<float, kWide>(master, i, n, p);
  if constexpr (sizeof(T) == 2) store_n<T, kWide>(static_cast<T*>(e.p), i, n, p);
  if constexpr (!k8) {
    store_n<float, kWide>(static_cast<float*>(e.m), i, n, m);
    store_n<float, kWide>(static_cast<float*>(e.v), i, n, v);
  } else {
    // a value that is no number spoils its own element and not its block: it takes no part in the scale and has the code of NaN
    float tm = 0, tv = 0;
#pragma unroll
    for (int k = 0; k < 8; k++) {
      v[k] = sqrtf(v[k]);
      if (fabsf(m[k]) <= 3.402823466e38f) tm = fmaxf(tm, fabsf(m[k]));
      if (v[k] <= 3.402823466e38f) tv = fmaxf(tv, v[k]);
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) {
      tm = fmaxf(tm, __shfl_xor_sync(0xffffffffu, tm, d));
      tv = fmaxf(tv, __shfl_xor_sync(0xffffffffu, tv, d));
    }
    const int em = scale_exponent(tm), ev = scale_exponent(tv);
    const float im = __uint_as_float((127 - em) << 23), iv = __uint_as_float((127 - ev) << 23);
    unsigned char a[8], b[8];
#pragma unroll
    for (int k = 0; k < 8; k++) {
      const unsigned u = random_bits(s.seed_mix, (unsigned long long)e.at * kBlock + (unsigned long long)(i + k));
      float q = copysignf(on_grid(fabsf(m[k]) * im, u & 0xffff), m[k]);
      a[k] = fabsf(m[k]) <= 3.402823466e38f ? code_of(q) : 0x7f;
      q = on_grid(v[k] * iv, u >> 16);
      if (v[k] > 0) q = fmaxf(q, 0.001953125f);
      b[k] = v[k] <= 3.402823466e38f ? code_of(q) : 0x7f;
    }
    store_codes<kWide>(mc, i, n, a);
    store_codes<kWide>(vc, i, n, b);
    if ((threadIdx.x & 31) == 0) {
      e.ms[block] = __uint_as_float((em + 127) << 23);
      e.vs[block] = __uint_as_float((ev + 127) << 23);
    }
  }
}

template <int N, bool k8>
__global__ void __launch_bounds__(kThreads) adamw_kernel(const __grid_constant__ Args<N> a) {
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

constexpr int kMost = 350;   // entries of 88 bytes in the 32764 bytes that a launch's parameters may have

__global__ void __launch_bounds__(kThreads) block8_values_kernel(__nv_bfloat16* __restrict__ out, const unsigned char* __restrict__ codes,
                                                                const float* __restrict__ scale, long long n, bool wide) {
  const long long i = ((long long)blockIdx.x * kThreads + threadIdx.x) * 8;
  if (i >= n) return;
  unsigned char c[8];
  float x[8];
  wide ? load_codes<true>(codes, i, n, c) : load_codes<false>(codes, i, n, c);
  const float s = scale[i / kBlock];
#pragma unroll
  for (int k = 0; k < 8; k++) x[k] = value_of(c[k]) * s;
  wide ? store_n<__nv_bfloat16, true>(out, i, n, x) : store_n<__nv_bfloat16, false>(out, i, n, x);
}

}  // namespace

int launch_adamw(int count, const gelib_adamw_tensor* t, const gelib_adamw_options& o, cudaStream_t stream) {
  Scalars s;
  const double c1 = 1 - std::pow(o.beta1, (double)o.step), c2 = 1 - std::pow(o.beta2, (double)o.step);
  s.b1 = (float)o.beta1, s.one_b1 = (float)(1 - o.beta1), s.b2 = (float)o.beta2, s.one_b2 = (float)(1 - o.beta2);
  s.keep = (float)(1 - o.lr * o.weight_decay), s.step = (float)(o.lr / c1), s.root = (float)(1 / std::sqrt(c2)), s.eps = (float)o.eps;
  s.grad_scale = o.grad_scale;
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
  const long long per = kThreads * 8, blocks = (n + per - 1) / per;
  if (blocks > 0x7fffffffLL) return fail(GELIB_INVALID, "block8_values", "too many elements");
  block8_values_kernel<<<(unsigned)blocks, kThreads, 0, stream>>>((__nv_bfloat16*)out, (const unsigned char*)codes, scale, n, wide);
  return launched("block8_values");
}

}  // namespace gelib_b200
