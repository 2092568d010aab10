// Operands as the tensor cores want them: float matrices as three bfloat16 planes, 16-bit ones with rows on 16-byte boundaries.
#pragma once
#include <algorithm>

#include "readout.h"
#include "linear.h"

namespace gelib_b200 {

namespace {

constexpr int kCopyThreads = 256;   // of a block that copies

long long up(long long bytes) { return (bytes + 255) / 256 * 256; }

// Operands to be copied: as three planes, or with rows on 16-byte boundaries.
struct PlaneJobs {
  Stored from[3];
  Stored to[3];
  long long first[4];   // number of a job's first chunk of eight columns; the last entry is the end
  int wide[3];          // rows begin on 16-byte boundaries
  int count;
  void add(const Stored& f, const Stored& t, int type) {
    from[count] = f, to[count] = t;
    wide[count] = is_aligned(f.base, 16) && f.ld * type_bytes(type) % 16 == 0;
    first[count + 1] = first[count] + (f.cols + 7) / 8 * f.rows;
    count++;
  }
};

// rows_out, where it is given: the rows r of the first operand with rows_out[r].y infinite become zero.  from: the first chunk that is copied.
template <class T, bool kOut = false>
__device__ __forceinline__ void copy_planes(const PlaneJobs& jobs, long long block, long long blocks, const float2* rows_out = nullptr, long long from = 0) {
  for (long long c = from + block * kCopyThreads + threadIdx.x; c < jobs.first[jobs.count]; c += blocks * kCopyThreads) {
    int job = 0;
    while (job + 1 < jobs.count && c >= jobs.first[job + 1]) job++;
    const Stored& f = jobs.from[job];
    const Stored& t = jobs.to[job];
    const long long chunks = (f.cols + 7) / 8, at = c - jobs.first[job], row = at / chunks, col = (at - row * chunks) * 8;
    const T* src = static_cast<const T*>(f.base) + row * f.ld + col;
    const int live = (int)min(8LL, f.cols - col);
    T x[8];
    if (jobs.wide[job] && live == 8) {
      constexpr int kLoads = sizeof(T) / 2;   // of 16 bytes
      union { uint4 u[kLoads]; T t[8]; } w;
#pragma unroll
      for (int i = 0; i < kLoads; i++) w.u[i] = reinterpret_cast<const uint4*>(src)[i];
#pragma unroll
      for (int j = 0; j < 8; j++) x[j] = w.t[j];
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++) x[j] = j < live ? src[j] : from_float<T>(0.f);
    }
    if constexpr (kOut)
      if (rows_out && job == 0 && rows_out[row].y == INFINITY)
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = from_float<T>(0.f);
    if constexpr (sizeof(T) == 4) {
      union { uint4 u; uint32_t t[4]; } w[3];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        uint32_t p[3];
        split3(x[2 * j], x[2 * j + 1], p);
#pragma unroll
        for (int i = 0; i < 3; i++) w[i].t[j] = p[i];
      }
#pragma unroll
      for (int i = 0; i < 3; i++) *reinterpret_cast<uint4*>((__nv_bfloat16*)t.base + i * t.plane + row * t.ld + col) = w[i].u;
    } else {
      union { uint4 u; T t[8]; } w;
#pragma unroll
      for (int j = 0; j < 8; j++) w.t[j] = x[j];
      *reinterpret_cast<uint4*>((T*)t.base + row * t.ld + col) = w.u;
    }
  }
}

long long planes_bytes(long long rows, long long cols, int type) { return up((cols + 7) / 8 * 8 * rows * (type == GELIB_F32 ? 6 : 2)); }
Stored planes_at(const Stored& s, int type, char*& at) {
  const long long ld = (s.cols + 7) / 8 * 8;
  const Stored to = {at, s.rows, s.cols, ld, s.rows * ld, type == GELIB_F32 ? 3 : 1};
  at += planes_bytes(s.rows, s.cols, type);
  return to;
}

// Bytes that an operand's copy takes, 0 where it is used as it lies.
long long copy_bytes(const Stored& s, int type) { return tc_ready(s, type) ? 0 : planes_bytes(s.rows, s.cols, type); }
void copy_if_needed(Stored* s, int type, char*& at, PlaneJobs* jobs) {
  if (tc_ready(*s, type)) return;
  const Stored to = planes_at(*s, type, at);
  jobs->add(*s, to, type);
  *s = to;
}

}  // namespace

}  // namespace gelib_b200
