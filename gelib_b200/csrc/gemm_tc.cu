// D = A B on the 5th-generation tensor cores, with the epilogue of a dense layer.
//
// A persistent block (or a pair of blocks on neighbouring SMs, which then share a tile of 256 rows and each hold half of B's columns) has two
// warps that bring 64-deep slabs of A and of B into a ring in shared memory by tensor copies, one that issues the multiplications, and eight
// that take finished sums out of tensor memory while the next tile is summed in its other half.  Either operand may lie
// with its rows along the sum or across it: the 128-byte swizzle serves both, and the instruction is told which.
//
// float matrices come as three bfloat16 planes a = a0 + a1 + a2; the six products a_i b_j with i + j <= 2 are summed, the rest is below 2^-22 of a product.
// A plane's slabs of A and B share a stage, so that a group of three stages carries the six.  The tensor cores cut every sum
// off at float's last bit instead of rounding it: over 1280 products in one accumulator the results were 9e-6 off, all to the same side.  So the
// five small products of a slab come first and a0 b0 last, and after every slab the sums leave tensor memory for registers, where
// they are added with rounding: four cuts at full size and no more (7e-7).
//
// Every wait has a limit; a kernel that gives up says so in a status word, and ends.
#include <cuda.h>

#include <algorithm>
#include <cmath>

#include "readout.h"
#include "linear.h"
#include "plan.h"
#include "tc_common.h"
#include "tma_maps.h"

namespace gelib_b200 {

namespace {

using tc::smem_u32;

constexpr int kDepth = 64;            // of a slab: 128 bytes of 16-bit numbers
constexpr int kSms = 148;
constexpr int kWarps = 8;              // that take the results: two for each quarter of tensor memory, which share a tile's columns
constexpr int kThreads = 96 + 32 * kWarps;   // beside two warps for copies and one for multiplications
constexpr int kChunk = 16;             // columns that such a warp takes at a time, every other chunk of the tile
constexpr int kPitch = kChunk + 4;     // floats of a staged row: 16-byte accesses by rows and by columns without conflicts
constexpr int kStaging = kWarps * 32 * kPitch * 4;

struct TcArgs {
  Epilogue e;
  float* part;                        // partial sums (splits, M, N), or null
  int* status;
  int limit;                          // of the first waits: kWaitLimit, or 0 where a test makes them run out
  long long M;
  int N;
  int slabs, per;                     // slabs of the sum, and of one split
  int splits, tiles_m, tiles_n;
  int bn;                             // columns of a tile
  int a_across, b_across;             // the operand's rows are the sum's index
  int bf16, vec;                      // operand type; columns may be taken four at a time
};

// A tile has 128 CG rows and up to kBnMost columns, a multiple of 16 (32 in a pair).
template <int CG, int P>
struct Shape {
  static constexpr int kBnMost = 128 * CG;
  static constexpr int kA = 128 * 128, kB = kBnMost / CG * 128;        // bytes of a slab in a block
  static constexpr int kStage = kA + kB;
  static constexpr int kStages = 6;                                    // a multiple of three
  static constexpr int kShared = kStages * kStage + kStaging + 1024;
};

struct Bars {
  uint64_t full[12], empty[12], sums_full[2], sums_empty[2], done;
  uint32_t tmem;
};

// The address of `local` in the shared memory of block `rank` of the cluster.
__device__ __forceinline__ uint32_t at_rank(uint32_t local, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(local), "r"(rank));
  return a;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// At most `limit` naps of a tenth of a millisecond; all lanes of a warp wait.
constexpr int kWaitLimit = 20000;
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, int limit = kWaitLimit) {
  const uint32_t a = smem_u32(bar);
  for (int i = 0; i < limit; i++) {
    uint32_t ok;
    asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3; selp.u32 %0, 1, 0, p; }"
                 : "=r"(ok)
                 : "r"(a), "r"(parity), "r"(100000u)
                 : "memory");
    if (ok) return true;
  }
  return false;
}
// Whether a phase is over now; asked ahead of other work, so that the answer is there when that is done.
__device__ __forceinline__ uint32_t over(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{ .reg .pred p; mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }" : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
  return ok;
}
__device__ __forceinline__ bool all_wait(uint64_t* bar, uint32_t parity, int limit = kWaitLimit) {
  return __all_sync(0xffffffffu, wait(bar, parity, limit));
}
// The copies, multiplications and their barriers below are issued by one elected lane of a converged warp: with a branch for lane 0 around the loop the
// compiler kept descriptors and addresses out of the uniform registers that these instructions take, and a slab's four multiplications
// took 240 cycles to issue, its two copies 210.
__device__ __forceinline__ void expect_bytes(uint64_t* bar, uint32_t bytes) {
  asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; @p mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1; }" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void arrive_at(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}

template <int CG>
__device__ __forceinline__ void copy_box(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  if constexpr (CG == 2)
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff;\n"
                 "@p cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, %4}], [%5]; }" ::"r"(dst),
                 "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
                 : "memory");
  else
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff;\n"
                 "@p cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5]; }" ::"r"(dst), "l"(map),
                 "r"(x), "r"(y), "r"(z), "r"(bar)
                 : "memory");
}

template <int CG>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  if constexpr (CG == 2)
    asm volatile("{ .reg .pred p, q; elect.sync _|p, 0xffffffff; setp.ne.b32 q, %4, 0; @p tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, q; }" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
                 "r"((uint32_t)accumulate)
                 : "memory");
  else
    asm volatile("{ .reg .pred p, q; elect.sync _|p, 0xffffffff; setp.ne.b32 q, %4, 0; @p tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, q; }" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
                 "r"((uint32_t)accumulate)
                 : "memory");
}
// Arrives on the barrier, in both blocks of a pair, when this thread's multiplications so far are done.
template <int CG>
__device__ __forceinline__ void commit(uint64_t* bar) {
  if constexpr (CG == 2)
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; @p tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1; }" ::"r"(smem_u32(bar)), "h"((uint16_t)3)
                 : "memory");
  else
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; @p tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0]; }" ::"r"(smem_u32(bar)) : "memory");
}

// Shared-memory descriptor of a slab, 128-byte swizzle.  Rows across the sum: 64 deep, eight rows of 128 bytes to a swizzle atom, atoms
// 1024 bytes apart.  Rows along the sum: blocks of 64 columns by 64 deep, 8192 bytes apart; eight deep to an atom.
__device__ __forceinline__ uint64_t slab_desc(uint32_t addr, bool across) {
  const uint64_t lead = across ? 8192 >> 4 : 1, step = 1024 >> 4;
  return (uint64_t)((addr & 0x3ffff) >> 4) | lead << 16 | step << 32 | 1ull << 46 | 2ull << 61;
}

struct Item {
  int m, n, split;
};
__device__ __forceinline__ Item item_of(const TcArgs& g, int i) {
  const int tiles = g.tiles_m * g.tiles_n, t = i % tiles;
  // groups of eight tiles of rows, so that the tiles at work at a time share operands in L2
  const int width = 8 * g.tiles_n, first = t / width * 8, high = min(8, g.tiles_m - first);
  return {first + t % width % high, t % width / high, i / tiles};
}

// A warp's 32 rows from m0 on of 16 columns from n0 on, a row per lane in r, through shared memory, so that lanes store along rows.
template <class T>
__device__ __forceinline__ void store_chunk(const TcArgs& g, int split, const uint32_t (&r)[kChunk], uint32_t block, long long m0, int n0, int lane, const float (&bias)[4]) {
  constexpr int kAcross = kChunk / 4, kRows = 32 / kAcross, kPasses = 32 / kRows;
  const int col = lane % kAcross * 4, n = n0 + col, live = min(4, g.N - n);
  const long long m = m0 + lane / kAcross;
  const T* residual = g.part ? nullptr : static_cast<const T*>(g.e.residual);
  __syncwarp();
#pragma unroll
  for (int j = 0; j < kAcross; j++) tc::sts128(block + (lane * kPitch + 4 * j) * 4, r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
  float add[kPasses][4];
#pragma unroll
  for (int pass = 0; pass < kPasses; pass++) {   // all of them asked for before the first is needed
    const long long at = (m + pass * kRows) * g.N + n;
#pragma unroll
    for (int j = 0; j < 4; j++) add[pass][j] = 0;
    if (residual && live > 0 && m + pass * kRows < g.M) {
      if (g.vec) load_vec<T, 4>(residual + at, add[pass]);
      else
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (j < live) add[pass][j] = to_float(residual[at + j]);
    }
  }
  __syncwarp();
#pragma unroll
  for (int pass = 0; pass < kPasses; pass++) {
    const float4 v = tc::lds128(block + ((pass * kRows + lane / kAcross) * kPitch + col) * 4);
    if (m + pass * kRows >= g.M || live <= 0) continue;
    float d[4] = {v.x, v.y, v.z, v.w};
    const long long at = (m + pass * kRows) * g.N + n;
    if (g.part) {
      float* p = g.part + (long long)split * g.M * g.N + at;
      if (g.vec) *reinterpret_cast<float4*>(p) = v;
      else
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (j < live) p[j] = d[j];
      continue;
    }
#pragma unroll
    for (int j = 0; j < 4; j++) d[j] += bias[j];
    if (g.e.z) {
      T q[4];
#pragma unroll
      for (int j = 0; j < 4; j++) q[j] = held<T>(d[j]);
      T* z = static_cast<T*>(g.e.z) + at;
      if (g.vec) {
        union { typename Raw<4 * sizeof(T)>::type raw; T t[4]; } w;
#pragma unroll
        for (int j = 0; j < 4; j++) w.t[j] = q[j];
        *reinterpret_cast<typename Raw<4 * sizeof(T)>::type*>(z) = w.raw;
      } else {
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (j < live) z[j] = q[j];
      }
    }
    activate(d, g.e.act);
#pragma unroll
    for (int j = 0; j < 4; j++) d[j] += add[pass][j];
    T* y = static_cast<T*>(g.e.y) + at;
    if (g.vec) store_vec<T, 4>(y, d);
    else
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (j < live) y[j] = from_float<T>(d[j]);
  }
}

// A lane's part of the bias in the chunk of columns from n0 on.
template <class T>
__device__ __forceinline__ void load_bias(const TcArgs& g, int n0, int lane, float (&bias)[4]) {
  const int n = n0 + lane % (kChunk / 4) * 4;
#pragma unroll
  for (int j = 0; j < 4; j++) bias[j] = g.e.bias && n + j < g.N ? to_float(static_cast<const T*>(g.e.bias)[n + j]) : 0.f;
}

template <class T, int CG, int P>
__global__ void __launch_bounds__(kThreads, 1) gemm_tc_kernel(const __grid_constant__ CUtensorMap ma, const __grid_constant__ CUtensorMap mb, TcArgs g) {
  using S = Shape<CG, P>;
  extern __shared__ unsigned char raw[];
  unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  __shared__ Bars bars;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;   // the compiler sees that a warp's lanes agree
  const uint32_t rank = CG == 2 ? blockIdx.x & 1 : 0;
  const int first = CG == 2 ? blockIdx.x >> 1 : blockIdx.x, stride = CG == 2 ? gridDim.x >> 1 : gridDim.x;
  const int items = g.tiles_m * g.tiles_n * g.splits;
  constexpr int kColumns = 2 * S::kBnMost;

  if (warp == 0 && lane == 0) {
    for (int i = 0; i < S::kStages; i++) tc::mbar_init(&bars.full[i], 2), tc::mbar_init(&bars.empty[i], 1);
    for (int i = 0; i < 2; i++) tc::mbar_init(&bars.sums_full[i], 1), tc::mbar_init(&bars.sums_empty[i], kWarps * CG);
    tc::mbar_init(&bars.done, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    if constexpr (CG == 2) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars.tmem)), "r"(kColumns) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars.tmem)), "r"(kColumns) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  tc::tc_fence_before();
  if constexpr (CG == 2) cluster_sync(); else __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = bars.tmem, ring_at = smem_u32(ring);
  bool ok = true;

  if (warp == 0 || warp == 2) {   // copies of A, of B
    const bool of_b = warp == 2, across = of_b ? g.b_across : g.a_across;
    const CUtensorMap* map = of_b ? &mb : &ma;
    const int mine = of_b ? g.bn / CG : 128, boxes = across ? (mine + 63) / 64 : 1;   // rows or columns in this block
    const uint32_t bytes = CG * (across ? boxes * 8192 : mine * 128), ring_mine = ring_at + (of_b ? S::kA : 0);
    int stage = 0;
    uint32_t phase = 0, ready = g.limit > 0 && over(&bars.empty[0], 1);
    long long issued = 0;
    for (int i = first; ok && i < items; i += stride) {
      const Item it = item_of(g, i);
      const int at = of_b ? it.n * g.bn + (int)rank * mine : (it.m * CG + (int)rank) * 128;
      const int k0 = it.split * g.per, k1 = min(g.slabs, k0 + g.per);
      for (int k = k0; ok && k < k1; k++)
        for (int p = 0; p < P; p++) {
          if (!__all_sync(0xffffffffu, ready) && !all_wait(&bars.empty[stage], phase ^ 1, g.limit)) {
            ok = false;
            break;
          }
          const uint32_t to = ring_mine + stage * S::kStage, full = smem_u32(&bars.full[stage]), bar = CG == 2 ? at_rank(full, 0) : full;
          if (rank == 0) expect_bytes(&bars.full[stage], bytes);
          if (++stage == S::kStages) stage = 0, phase ^= 1;
          ready = over(&bars.empty[stage], phase ^ 1);
          if (across)
            for (int j = 0; j < boxes; j++) copy_box<CG>(to + j * 8192, map, at + j * 64, k * kDepth, p, bar);
          else
            copy_box<CG>(to, map, k * kDepth, at, p, bar);
          issued++;
        }
    }
    if (!ok && rank == 0)   // copies in flight land before the block ends
      for (int i = 0; i < S::kStages && i < issued; i++) {
        const long long n = (issued - 1 - i) / S::kStages;   // how often stage i was filled before its last time
        wait(&bars.full[i], (uint32_t)(n & 1));
      }
  } else if (warp == 1 && rank == 0) {
    const uint32_t type = g.bf16 ? 1u : 0u;
    const uint32_t idesc = 1u << 4 | type << 7 | type << 10 | (uint32_t)g.a_across << 15 | (uint32_t)g.b_across << 16 | (uint32_t)(g.bn >> 3) << 17 | ((128u * CG) >> 4) << 24;
    // 16 deep further: 32 bytes along a row, or two atoms of eight rows
    const uint32_t step_a = (g.a_across ? 2048 : 32) >> 4, step_b = (g.b_across ? 2048 : 32) >> 4;
    int stage = 0, buf = 0;
    uint32_t phase = 0, buf_phase = 0, ready = 0;
    for (int i = first; ok && i < items; i += stride) {
      const Item it = item_of(g, i);
      const int k0 = it.split * g.per, k1 = min(g.slabs, k0 + g.per);
      bool more = false;
      auto slab = [&](int sa, int sb) {
        const uint64_t a = slab_desc(ring_at + sa * S::kStage, g.a_across), b = slab_desc(ring_at + sb * S::kStage + S::kA, g.b_across);
#pragma unroll
        for (int q = 0; q < kDepth / 16; q++) {
          mma<CG>(tmem + buf * S::kBnMost, a + q * step_a, b + q * step_b, idesc, more);
          more = true;
        }
      };
      auto begin = [&] {
        if (!(ok = all_wait(&bars.sums_empty[buf], buf_phase ^ 1, g.limit))) return false;
        tc::tc_fence_after();
        more = false;
        return true;
      };
      auto end = [&] {
        commit<CG>(&bars.sums_full[buf]);
        buf ^= 1;
        if (buf == 0) buf_phase ^= 1;
      };
      auto arrived = [&](int s) {
        ok = __all_sync(0xffffffffu, ready) || all_wait(&bars.full[s], phase);
        ready = 0;
        tc::tc_fence_after();
        return ok;
      };
      if constexpr (P == 1) {
        if (!begin()) break;
        for (int k = k0; k < k1; k++) {
          if (!arrived(stage)) break;
          const int now = stage;
          if (++stage == S::kStages) stage = 0, phase ^= 1;
          ready = over(&bars.full[stage], phase);
          slab(now, now);
          commit<CG>(&bars.empty[now]);
        }
        end();
      } else {
        for (int k = k0; k < k1; k++) {   // three stages of a turn: the ring has a multiple of three
          const int s = stage;
          if (!begin() || !arrived(s) || !arrived(s + 1)) break;
          slab(s + 1, s + 1);
          slab(s + 1, s);
          slab(s, s + 1);
          commit<CG>(&bars.empty[s + 1]);
          if (!arrived(s + 2)) break;
          slab(s + 2, s);
          slab(s, s + 2);
          commit<CG>(&bars.empty[s + 2]);
          slab(s, s);
          commit<CG>(&bars.empty[s]);
          end();
          stage += 3;
          if (stage == S::kStages) stage = 0, phase ^= 1;
        }
      }
    }
    if (!ok) {   // what was issued ends before tensor memory is given back
      commit<CG>(&bars.done);
      wait(&bars.done, 0);
    }
  } else if (warp >= 3) {
    const int q = warp & 3;                          // the quarter of tensor memory that the warp may read
    const int mine = (warp - 3) / 4 * kChunk;        // its first chunk
    const uint32_t block = ring_at + S::kStages * S::kStage + (warp - 3) * 32 * kPitch * 4;
    constexpr int kChunks = S::kBnMost / (2 * kChunk);   // at most
    int buf = 0;
    uint32_t buf_phase = 0;
    auto taken = [&] {   // tensor memory has been read
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_at(at_rank(smem_u32(&bars.sums_empty[buf]), 0));
      buf ^= 1;
      if (buf == 0) buf_phase ^= 1;
    };
    for (int i = first; ok && i < items; i += stride) {
      const Item it = item_of(g, i);
      const long long m0 = ((long long)it.m * CG + rank) * 128 + q * 32;
      const int n0 = it.n * g.bn + mine;
      const uint32_t from = tmem + ((uint32_t)q << 21) + mine;
      auto has = [&](int c) { return mine + c * 2 * kChunk < g.bn && n0 + c * 2 * kChunk < g.N; };
      float bias[P == 1 ? kChunks : 1][4];
      if constexpr (P == 1) {
#pragma unroll
        for (int c = 0; c < kChunks; c++) load_bias<T>(g, n0 + c * 2 * kChunk, lane, bias[c]);
        if (!(ok = all_wait(&bars.sums_full[buf], buf_phase, g.limit))) break;
        tc::tc_fence_after();
#pragma unroll
        for (int c = 0; c < kChunks; c++)
          if (has(c)) {
            uint32_t r[kChunk];
            tc::tmem_ld16(from + buf * S::kBnMost + c * 2 * kChunk, r);
            store_chunk<T>(g, it.split, r, block, m0, n0 + c * 2 * kChunk, lane, bias[c]);
          }
        taken();
      } else {
        float sum[kChunks][kChunk];
#pragma unroll
        for (int c = 0; c < kChunks; c++)
#pragma unroll
          for (int j = 0; j < kChunk; j++) sum[c][j] = 0;
        const int k0 = it.split * g.per, k1 = min(g.slabs, k0 + g.per);
        for (int k = k0; k < k1; k++) {
          if (!(ok = all_wait(&bars.sums_full[buf], buf_phase, g.limit))) break;
          tc::tc_fence_after();
#pragma unroll
          for (int c = 0; c < kChunks; c++)
            if (has(c)) {
              uint32_t r[kChunk];
              tc::tmem_ld16(from + buf * S::kBnMost + c * 2 * kChunk, r);
#pragma unroll
              for (int j = 0; j < kChunk; j++) sum[c][j] += __uint_as_float(r[j]);
            }
          taken();
        }
        if (!ok) break;
#pragma unroll
        for (int c = 0; c < kChunks; c++)
          if (has(c)) {
            load_bias<T>(g, n0 + c * 2 * kChunk, lane, bias[0]);
            uint32_t r[kChunk];
#pragma unroll
            for (int j = 0; j < kChunk; j++) r[j] = __float_as_uint(sum[c][j]);
            store_chunk<T>(g, it.split, r, block, m0, n0 + c * 2 * kChunk, lane, bias[0]);
          }
      }
    }
  }
  if (!ok && g.status) *reinterpret_cast<volatile int*>(g.status) = 1;
  __syncwarp();
  tc::tc_fence_before();
  if constexpr (CG == 2) cluster_sync(); else __syncthreads();
  tc::tc_fence_after();
  if (warp == 1) {
    if constexpr (CG == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kColumns) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kColumns) : "memory");
  }
}

// ---- operands as the kernel wants them ----------------------------------------------------------------------------------------------

struct PlaneJobs {
  Stored from[3];
  void* to[3];
  long long first[4];   // number of a job's first chunk of eight columns; the last entry is the end
  int wide[3];          // rows begin on 16-byte boundaries
  int count;
};

template <class T>
__global__ void __launch_bounds__(256) planes_kernel(const __grid_constant__ PlaneJobs jobs) {
  for (long long c = (long long)blockIdx.x * 256 + threadIdx.x; c < jobs.first[jobs.count]; c += (long long)gridDim.x * 256) {
    int job = 0;
    while (job + 1 < jobs.count && c >= jobs.first[job + 1]) job++;
    const Stored& f = jobs.from[job];
    const long long chunks = (f.cols + 7) / 8, at = c - jobs.first[job], row = at / chunks, col = (at - row * chunks) * 8;
    const T* src = static_cast<const T*>(f.base) + row * f.ld + col;
    const int live = (int)min(8LL, f.cols - col);
    const long long ld = chunks * 8;
    if constexpr (sizeof(T) == 4) {
      float x[8];
      if (jobs.wide[job] && live == 8) {
        const float4 u = *reinterpret_cast<const float4*>(src), v = *reinterpret_cast<const float4*>(src + 4);
        x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w, x[4] = v.x, x[5] = v.y, x[6] = v.z, x[7] = v.w;
      } else {
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = j < live ? src[j] : 0.f;
      }
      union { uint4 u; __nv_bfloat16 t[8]; } w[3];
#pragma unroll
      for (int j = 0; j < 8; j++) {
        __nv_bfloat16 p[3];
        split3(x[j], p);
#pragma unroll
        for (int i = 0; i < 3; i++) w[i].t[j] = p[i];
      }
#pragma unroll
      for (int i = 0; i < 3; i++) *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(jobs.to[job]) + i * f.rows * ld + row * ld + col) = w[i].u;
    } else {
      union { uint4 u; T t[8]; } w;
#pragma unroll
      for (int j = 0; j < 8; j++) w.t[j] = j < live ? src[j] : from_float<T>(0.f);
      *reinterpret_cast<uint4*>(static_cast<T*>(jobs.to[job]) + row * ld + col) = w.u;
    }
  }
}

// ---- host -----------------------------------------------------------------------------------------------------------------------------

struct Config {
  int cg, bn, splits;
};

// The tile and the number of splits with the least estimated time, in microseconds.  Measured of a slab 64 deep, with every SM at work
// (4096 x 7168 x 2048): a pair's tile of 64, 128, 160, 192, 224, 256 columns 0.20, 0.24, 0.28, 0.29, 0.31, 0.40, a block's of 64, 128 0.20, 0.24;
// in float (4096 x 4096 x 4096) a pair's of 64, 128, 256 1.4, 1.7, 2.3, a block's of 32, 64, 128 1.2, 1.3, 1.5.
Config choose_config(long long M, long long N, long long K, int type) {
  const long long slabs = (K + kDepth - 1) / kDepth;
  Config best = {1, 128, 1};
  double best_time = 1e30;
  for (int cg = 1; cg <= 2; cg++)
    for (int bn = 128 * cg; bn >= 32 * cg; bn -= 16 * cg) {
      if (bn > 32 * cg && (N + bn - 1) / bn == (N + bn - 16 * cg - 1) / (bn - 16 * cg)) continue;   // a narrower tile covers N as often
      const long long tiles = ((M + 128 * cg - 1) / (128 * cg)) * ((N + bn - 1) / bn);
      const int slots = kSms / cg;
      const double slab = type == GELIB_F32 ? 1.15 + bn * (cg == 2 ? 0.0044 : 0.0031) : cg == 2 ? 0.13 + bn * 0.00101 : 0.16 + bn * 0.00064;
      for (int splits = 1; splits <= 64 && splits <= slabs; splits++) {
        if (splits > 1 && (tiles * splits > 4 * slots || slabs / splits < 4)) break;
        const long long per = (slabs + splits - 1) / splits;
        const double waves = std::ceil((double)tiles * splits / slots), results = 0.6 + bn * (cg == 2 ? 0.012 : 0.01);
        // a tile's results leave while the next is summed; the last one's do not
        double time = 2 + waves * std::max(per * slab, results) + results;
        if (splits > 1) time += 2.5 + (double)(splits + 1) * M * N * 4 / 4e6;
        if (time < best_time) best_time = time, best = {cg, bn, (int)((slabs + per - 1) / per)};
      }
    }
  return best;
}

bool encode(CUtensorMap* map, const Stored& s, int type, int box_x, int box_y) {
  EncodeTiledFn enc = encode_tiled();
  if (!enc) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)s.cols, (cuuint64_t)s.rows, (cuuint64_t)s.planes};
  const cuuint64_t line = (cuuint64_t)(s.rows > 1 ? s.ld : (s.cols + 7) / 8 * 8) * 2;
  const cuuint64_t strides[2] = {line, s.planes > 1 ? (cuuint64_t)s.plane * 2 : line * (cuuint64_t)s.rows};
  const cuuint32_t box[3] = {(cuuint32_t)box_x, (cuuint32_t)box_y, 1}, one[3] = {1, 1, 1};
  if (dims[0] > 0xffffffffULL || dims[1] > 0xffffffffULL || strides[0] >= 1ULL << 40 || strides[1] >= 1ULL << 40) return false;
  return enc(map, type == GELIB_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(s.base), dims, strides, box, one,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class T, int CG, int P>
int launch_as(const CUtensorMap& ma, const CUtensorMap& mb, const TcArgs& a, cudaStream_t stream) {
  static const char* fn = "linear";
  auto kernel = gemm_tc_kernel<T, CG, P>;
  constexpr int shared = Shape<CG, P>::kShared;
  GELIB_CUDA_TRY(fn, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, shared));
  const long long items = (long long)a.tiles_m * a.tiles_n * a.splits;
  cudaLaunchConfig_t c = {};
  c.gridDim = dim3((unsigned)std::min<long long>(items, kSms / CG) * CG);
  c.blockDim = dim3(kThreads);
  c.dynamicSmemBytes = shared;
  c.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = CG, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
  c.attrs = at;
  c.numAttrs = CG > 1 ? 1 : 0;
  GELIB_CUDA_TRY(fn, cudaLaunchKernelEx(&c, kernel, ma, mb, a));
  return launched(fn);
}

template <class T, int P>
int launch_config(const Config& c, const CUtensorMap& ma, const CUtensorMap& mb, const TcArgs& a, cudaStream_t stream) {
  return c.cg == 2 ? launch_as<T, 2, P>(ma, mb, a, stream) : launch_as<T, 1, P>(ma, mb, a, stream);
}

}  // namespace

bool tc_ready(const Stored& s, int type) {
  if (type == GELIB_F32 && s.planes != 3) return false;
  return is_aligned(s.base, 16) && (s.rows <= 1 || s.ld % 8 == 0);
}

long long planes_bytes(long long rows, long long cols, int type) { return (cols + 7) / 8 * 8 * rows * (type == GELIB_F32 ? 6 : 2); }

Stored planes_of(const Stored& s, int type, void* memory) {
  const long long ld = (s.cols + 7) / 8 * 8;
  return {memory, s.rows, s.cols, ld, s.rows * ld, type == GELIB_F32 ? 3 : 1};
}

int launch_planes(const Stored* from, const Stored* to, int count, int type, cudaStream_t stream) {
  PlaneJobs jobs = {};
  long long chunks = 0;
  for (int i = 0; i < count; i++) {
    jobs.from[i] = from[i];
    jobs.to[i] = const_cast<void*>(to[i].base);
    jobs.wide[i] = is_aligned(from[i].base, 16) && from[i].ld * type_bytes(type) % 16 == 0;
    jobs.first[i] = chunks;
    chunks += (from[i].cols + 7) / 8 * from[i].rows;
  }
  jobs.first[count] = chunks;
  jobs.count = count;
  if (chunks == 0) return GELIB_OK;
  const unsigned blocks = (unsigned)std::min((chunks + 255) / 256, (long long)kSms * 16);
  if (type == GELIB_F32) planes_kernel<float><<<blocks, 256, 0, stream>>>(jobs);
  else if (type == GELIB_BF16) planes_kernel<__nv_bfloat16><<<blocks, 256, 0, stream>>>(jobs);
  else planes_kernel<__half><<<blocks, 256, 0, stream>>>(jobs);
  return launched("linear");
}

long long tc_gemm_workspace(long long M, long long N, long long K, int type) {
  const Config c = choose_config(M, N, K, type);
  return c.splits > 1 ? (long long)c.splits * M * N * 4 : 0;
}

int launch_tc_gemm(const Gemm& g, void* workspace, cudaStream_t stream) {
  static const char* fn = "linear";
  const Config c = choose_config(g.M, g.N, g.K, g.type);
  CUtensorMap ma, mb;
  // rows across the sum: 64 deep and a tile's rows; rows along it: 64 columns and 64 deep
  if (!encode(&ma, g.a.s, g.type, 64, g.a.by_sum ? 64 : 128) || !encode(&mb, g.b.s, g.type, 64, g.b.by_sum ? 64 : c.bn / c.cg))
    return fail(GELIB_CUDA_ERROR, fn, "a tensor map could not be made");
  TcArgs a = {};
  a.e = g.e;
  a.part = c.splits > 1 ? (float*)workspace : nullptr;
  a.status = async_status_word(kStatusGemmTc);
  a.limit = inject_timeout() ? 0 : kWaitLimit;
  a.M = g.M, a.N = (int)g.N;
  a.slabs = (int)((g.K + kDepth - 1) / kDepth);
  a.per = (a.slabs + c.splits - 1) / c.splits;
  a.splits = c.splits;
  const long long tm = (g.M + 128 * c.cg - 1) / (128 * c.cg), tn = (g.N + c.bn - 1) / c.bn;
  if (tm * tn * c.splits > 0x3fffffffLL) return fail(GELIB_INVALID, fn, "too many elements");
  a.tiles_m = (int)tm, a.tiles_n = (int)tn;
  a.bn = c.bn;
  a.a_across = g.a.by_sum, a.b_across = g.b.by_sum;
  a.bf16 = g.type != GELIB_F16;
  const int four = 4 * type_bytes(g.type);
  a.vec = g.N % 4 == 0 && is_aligned(g.e.y, four) && is_aligned(g.e.z, four) && is_aligned(g.e.residual, four);
  int st;
  if (g.type == GELIB_F32) st = launch_config<float, 3>(c, ma, mb, a, stream);
  else if (g.type == GELIB_BF16) st = launch_config<__nv_bfloat16, 1>(c, ma, mb, a, stream);
  else st = launch_config<__half, 1>(c, ma, mb, a, stream);
  if (st != GELIB_OK || !a.part) return st;
  return launch_join(g, a.part, c.splits, stream);
}

}  // namespace gelib_b200
