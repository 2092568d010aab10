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
// they are added with rounding: four cuts at full size and no more (1.9e-7; the library's float product 7e-7).
//
// What bounds it: bfloat16, 4096 x 7168 x 2048 83 us (1440 TFLOP/s; the library 80), where 128 tiles on 74 pairs are two rounds; 8192^3 690 us (1600; the
// library 660).  A pair's slab for a tile of 256 columns takes 0.38 us, its multiplications 0.27: the rest is the slabs' way out of L2.  Sums of 1152 are short beside
// the epilogue: 16384 x 1152 x 1152 62 us, the library 53.  float, 4096^3 650 us (210 TFLOP/s of float products, six times as many on the tensor cores).
// Steps, first size in tiles of 128 x 128: one lane issuing in a branch 138 us, an elected lane of a converged warp 117, one warp for A and one for B 105.
//
// Every wait has a limit; a kernel that gives up says so in a status word, and ends.
#include <cuda.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <map>
#include <mutex>
#include <vector>

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

// One product of a launch.
struct TcProblem {
  Epilogue e;
  float* part;                        // partial sums (splits, M, N), or null
  long long M;
  int N;
  int slabs, per;                     // slabs of the sum, and of one split
  int splits, tiles_m, tiles_n, items;
  int bn;                             // columns of a tile
  int a_across, b_across;             // the operand's rows are the sum's index
  int vec;                            // columns may be taken four at a time
};
constexpr int kProblems = 2;
struct TcArgs {
  TcProblem p[kProblems];             // those with longer items first
  int items;                          // of all
  int flip;                           // every other round of items is handed out from the last block on
  int* status;
  int limit;                          // of the first waits: kWaitLimit, or 0 where a test makes them run out
  int bf16;
};
struct TcMaps {
  CUtensorMap a[kProblems], b[kProblems];
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
  int m, n, split, k0, k1;
};
__device__ __forceinline__ Item item_of(const TcProblem& g, int i) {
  const int tiles = g.tiles_m * g.tiles_n, t = i % tiles, split = i / tiles;
  // groups of eight tiles of rows, so that the tiles at work at a time share operands in L2
  const int width = 8 * g.tiles_n, first = t / width * 8, high = min(8, g.tiles_m - first);
  return {first + t % width % high, t % width / high, split, split * g.per, min(g.slabs, (split + 1) * g.per)};
}

// The items of a block (or pair) in their order: item `at` of problem `which`, until there are no more.
struct Walk {
  int round, at, which;
  __device__ __forceinline__ bool next(const TcArgs& a, int mine, int blocks) {
    at = round * blocks + (a.flip && (round & 1) ? blocks - 1 - mine : mine);
    round++;
    if (at >= a.items) return false;
    which = at >= a.p[0].items;
    if (which) at -= a.p[0].items;
    return true;
  }
};

constexpr int kAcross = kChunk / 4, kRows = 32 / kAcross, kPasses = 32 / kRows;

// A lane's part of the residual in the warp's 32 rows from m0 on of 16 columns from n0 on, as it lies.
template <class T>
struct Rest {
  typename Raw<4 * sizeof(T)>::type raw[kPasses];
};
template <class T>
__device__ __forceinline__ void load_rest(const TcProblem& g, long long m0, int n0, int lane, Rest<T>& rest) {
  const T* residual = static_cast<const T*>(g.e.residual);
  if (!residual || g.part) return;
  const int n = n0 + lane % kAcross * 4;
#pragma unroll
  for (int pass = 0; pass < kPasses; pass++) {
    const long long m = m0 + pass * kRows + lane / kAcross, at = m * g.N + n;
    if (m < g.M && n < g.N) {
      if (g.vec) rest.raw[pass] = *reinterpret_cast<const typename Raw<4 * sizeof(T)>::type*>(residual + at);
      else {
        union { typename Raw<4 * sizeof(T)>::type raw; T t[4]; } w;
#pragma unroll
        for (int j = 0; j < 4; j++) w.t[j] = n + j < g.N ? residual[at + j] : from_float<T>(0.f);
        rest.raw[pass] = w.raw;
      }
    }
  }
}

// Those rows and columns, a row per lane in r, through shared memory, so that lanes store along rows.
template <class T>
__device__ __forceinline__ void store_chunk(const TcProblem& g, int split, const uint32_t (&r)[kChunk], uint32_t block, long long m0, int n0, int lane, const float (&bias)[4],
                                            const Rest<T>& rest) {
  const int col = lane % kAcross * 4, n = n0 + col, live = min(4, g.N - n);
  const long long m = m0 + lane / kAcross;
  __syncwarp();
#pragma unroll
  for (int j = 0; j < kAcross; j++) tc::sts128(block + (lane * kPitch + 4 * j) * 4, r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
  __syncwarp();
  if (g.vec && m0 + 32 <= g.M && n0 + kChunk <= g.N) {
    // nothing to be left out: all sixteen sums of the lane go through each step together
    float d[kPasses][4];
#pragma unroll
    for (int pass = 0; pass < kPasses; pass++) {
      const float4 v = tc::lds128(block + ((pass * kRows + lane / kAcross) * kPitch + col) * 4);
      d[pass][0] = v.x, d[pass][1] = v.y, d[pass][2] = v.z, d[pass][3] = v.w;
    }
    const long long at = m * g.N + n, step = (long long)kRows * g.N;
    if (g.part) {
      float* p = g.part + (long long)split * g.M * g.N + at;
#pragma unroll
      for (int pass = 0; pass < kPasses; pass++) store_vec<float, 4>(p + pass * step, d[pass]);
      return;
    }
#pragma unroll
    for (int pass = 0; pass < kPasses; pass++)
#pragma unroll
      for (int j = 0; j < 4; j++) d[pass][j] += bias[j];
    if (g.e.z) {
      T* z = static_cast<T*>(g.e.z) + at;
#pragma unroll
      for (int pass = 0; pass < kPasses; pass++) {
        union { typename Raw<4 * sizeof(T)>::type raw; T t[4]; } w;
#pragma unroll
        for (int j = 0; j < 4; j++) w.t[j] = held<T>(d[pass][j]);
        *reinterpret_cast<typename Raw<4 * sizeof(T)>::type*>(z + pass * step) = w.raw;
      }
    }
    activate(reinterpret_cast<float(&)[4 * kPasses]>(d), g.e.act);
    if (g.e.residual)
#pragma unroll
      for (int pass = 0; pass < kPasses; pass++) {
        union { typename Raw<4 * sizeof(T)>::type raw; T t[4]; } w;
        w.raw = rest.raw[pass];
#pragma unroll
        for (int j = 0; j < 4; j++) d[pass][j] += to_float(w.t[j]);
      }
    T* y = static_cast<T*>(g.e.y) + at;
#pragma unroll
    for (int pass = 0; pass < kPasses; pass++) store_vec<T, 4>(y + pass * step, d[pass]);
    return;
  }
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
    union { typename Raw<4 * sizeof(T)>::type raw; T t[4]; } w;
    if (g.e.z) {
#pragma unroll
      for (int j = 0; j < 4; j++) w.t[j] = held<T>(d[j]);
      T* z = static_cast<T*>(g.e.z) + at;
      if (g.vec) *reinterpret_cast<typename Raw<4 * sizeof(T)>::type*>(z) = w.raw;
      else
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (j < live) z[j] = w.t[j];
    }
    activate(d, g.e.act);
    if (g.e.residual) {
      w.raw = rest.raw[pass];
#pragma unroll
      for (int j = 0; j < 4; j++) d[j] += to_float(w.t[j]);
    }
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
__device__ __forceinline__ void load_bias(const TcProblem& g, int n0, int lane, float (&bias)[4]) {
  const int n = n0 + lane % kAcross * 4;
#pragma unroll
  for (int j = 0; j < 4; j++) bias[j] = g.e.bias && n + j < g.N ? to_float(static_cast<const T*>(g.e.bias)[n + j]) : 0.f;
}

template <class T, int CG, int P>
__global__ void __launch_bounds__(kThreads, 1) gemm_tc_kernel(const __grid_constant__ TcMaps maps, const __grid_constant__ TcArgs args) {
  using S = Shape<CG, P>;
  extern __shared__ unsigned char raw[];
  unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  __shared__ Bars bars;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;   // the compiler sees that a warp's lanes agree
  const uint32_t rank = CG == 2 ? blockIdx.x & 1 : 0;
  const int mine_of = CG == 2 ? blockIdx.x >> 1 : blockIdx.x, blocks = CG == 2 ? gridDim.x >> 1 : gridDim.x;
  Walk walk = {0, 0, 0};
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
  let_next_begin();
  await_previous();

  if (warp == 0 || warp == 2) {   // copies of A, of B
    const bool of_b = warp == 2;
    const uint32_t ring_mine = ring_at + (of_b ? S::kA : 0);
    int stage = 0;
    uint32_t phase = 0, ready = args.limit > 0 && over(&bars.empty[0], 1);
    long long issued = 0;
    while (ok && walk.next(args, mine_of, blocks)) {
      const TcProblem& g = args.p[walk.which];
      const Item it = item_of(g, walk.at);
      const bool across = of_b ? g.b_across : g.a_across;
      const CUtensorMap* map = of_b ? &maps.b[walk.which] : &maps.a[walk.which];
      const int mine = of_b ? g.bn / CG : 128, boxes = across ? (mine + 63) / 64 : 1;   // rows or columns in this block
      const uint32_t bytes = CG * (across ? boxes * 8192 : mine * 128);
      const int at = of_b ? it.n * g.bn + (int)rank * mine : (it.m * CG + (int)rank) * 128;
      const int k0 = it.k0, k1 = it.k1;
      for (int k = k0; ok && k < k1; k++)
        for (int p = 0; p < P; p++) {
          if (!__all_sync(0xffffffffu, ready) && !all_wait(&bars.empty[stage], phase ^ 1, args.limit)) {
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
    const uint32_t type = args.bf16 ? 1u : 0u;
    int stage = 0, buf = 0;
    uint32_t phase = 0, buf_phase = 0, ready = 0;
    while (ok && walk.next(args, mine_of, blocks)) {
      const TcProblem& g = args.p[walk.which];
      const Item it = item_of(g, walk.at);
      const int k0 = it.k0, k1 = it.k1;
      const uint32_t a_across = g.a_across, b_across = g.b_across;
      const uint32_t idesc = 1u << 4 | type << 7 | type << 10 | a_across << 15 | b_across << 16 | (uint32_t)(g.bn >> 3) << 17 | ((128u * CG) >> 4) << 24;
      // 16 deep further: 32 bytes along a row, or two atoms of eight rows
      const uint32_t step_a = (a_across ? 2048 : 32) >> 4, step_b = (b_across ? 2048 : 32) >> 4;
      bool more = false;
      auto slab = [&](int sa, int sb) {
        const uint64_t a = slab_desc(ring_at + sa * S::kStage, a_across), b = slab_desc(ring_at + sb * S::kStage + S::kA, b_across);
#pragma unroll
        for (int q = 0; q < kDepth / 16; q++) {
          mma<CG>(tmem + buf * S::kBnMost, a + q * step_a, b + q * step_b, idesc, more);
          more = true;
        }
      };
      auto begin = [&] {
        if (!(ok = all_wait(&bars.sums_empty[buf], buf_phase ^ 1, args.limit))) return false;
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
    while (ok && walk.next(args, mine_of, blocks)) {
      const TcProblem g = walk.which ? args.p[1] : args.p[0];   // in registers: the choice costs a load at every use otherwise
      const Item it = item_of(g, walk.at);
      const long long m0 = ((long long)it.m * CG + rank) * 128 + q * 32;
      const int n0 = it.n * g.bn + mine;
      const uint32_t from = tmem + ((uint32_t)q << 21) + mine;
      auto has = [&](int c) { return mine + c * 2 * kChunk < g.bn && n0 + c * 2 * kChunk < g.N; };
      Rest<T> rest[2];   // of a chunk, and of the next, asked for before the first is stored
      auto store = [&](int c, const uint32_t (&r)[kChunk], const float (&bias)[4]) {
        if (c + 1 < kChunks && has(c + 1)) load_rest<T>(g, m0, n0 + (c + 1) * 2 * kChunk, lane, rest[(c + 1) & 1]);
        store_chunk<T>(g, it.split, r, block, m0, n0 + c * 2 * kChunk, lane, bias, rest[c & 1]);
      };
      if constexpr (P == 1) {
        float bias[kChunks][4];
#pragma unroll
        for (int c = 0; c < kChunks; c++) load_bias<T>(g, n0 + c * 2 * kChunk, lane, bias[c]);
        load_rest<T>(g, m0, n0, lane, rest[0]);
        if (!(ok = all_wait(&bars.sums_full[buf], buf_phase, args.limit))) break;
        tc::tc_fence_after();
#pragma unroll
        for (int c = 0; c < kChunks; c++)
          if (has(c)) {
            uint32_t r[kChunk];
            tc::tmem_ld16(from + buf * S::kBnMost + c * 2 * kChunk, r);
            store(c, r, bias[c]);
          }
        taken();
      } else {
        float sum[kChunks][kChunk];
#pragma unroll
        for (int c = 0; c < kChunks; c++)
#pragma unroll
          for (int j = 0; j < kChunk; j++) sum[c][j] = 0;
        for (int k = it.k0; k < it.k1; k++) {
          if (!(ok = all_wait(&bars.sums_full[buf], buf_phase, args.limit))) break;
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
        load_rest<T>(g, m0, n0, lane, rest[0]);
#pragma unroll
        for (int c = 0; c < kChunks; c++)
          if (has(c)) {
            float bias[4];
            load_bias<T>(g, n0 + c * 2 * kChunk, lane, bias);
            uint32_t r[kChunk];
#pragma unroll
            for (int j = 0; j < kChunk; j++) r[j] = __float_as_uint(sum[c][j]);
            store(c, r, bias);
          }
      }
    }
  }
  if (!ok && args.status) *reinterpret_cast<volatile int*>(args.status) = 1;
  __syncwarp();
  tc::tc_fence_before();
  if constexpr (CG == 2) cluster_sync(); else __syncthreads();
  tc::tc_fence_after();
  if (warp == 1) {
    if constexpr (CG == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kColumns) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kColumns) : "memory");
  }
}

// ---- host -----------------------------------------------------------------------------------------------------------------------------

struct Config {
  int bn, splits;
};
struct Plan {
  int cg, flip;
  Config c[kProblems];
};
struct Sizes {
  long long M, N, K;
};

// Estimates in microseconds.  Measured of a slab 64 deep, with every SM at work (4096 x 7168 x 2048): a pair's tile of 64, 128, 160, 192, 224, 256
// columns 0.20, 0.24, 0.28, 0.29, 0.31, 0.40, a block's of 64, 128 0.20, 0.24; in float (4096 x 4096 x 4096) a pair's of 64, 128, 256 1.4,
// 1.7, 2.3, a block's of 32, 64, 128 1.2, 1.3, 1.5.
double slab_time(int cg, int bn, int type) {
  if (type == GELIB_F32) return 1.15 + bn * (cg == 2 ? 0.0044 : 0.0031);
  return cg == 2 ? 0.13 + bn * 0.00101 : 0.16 + bn * 0.00064;
}

struct Work {
  double items, each;   // how many, and the time of one
  double join;          // of the partial sums
};
Work work_of(const Sizes& z, int cg, const Config& c, int type) {
  const long long slabs = (z.K + kDepth - 1) / kDepth, per = (slabs + c.splits - 1) / c.splits;
  const double items = (double)((z.M + 128 * cg - 1) / (128 * cg)) * ((z.N + c.bn - 1) / c.bn) * c.splits;
  // a tile's results leave while the next is summed, if that takes as long
  const double results = 0.6 + c.bn * (cg == 2 ? 0.012 : 0.01);
  return {items, std::max(per * slab_time(cg, c.bn, type), results), c.splits > 1 ? (double)(c.splits + 1) * z.M * z.N * 4 / 4e6 : 0};
}

// The time of a launch of one or two products, whose items are handed out round by round, longer ones first.
double launch_time(const Work* w, int count, int slots) {
  double join = 0, all = 0, most = 0, items = 0, least = 1e30;
  for (int i = 0; i < count; i++) {
    join += w[i].join, all += w[i].items * w[i].each, items += w[i].items;
    most = std::max(most, w[i].each), least = std::min(least, w[i].each);
  }
  const double rounds = std::ceil(items / slots);
  // with one kind of item whole rounds; with two the shorter ones fill in
  const double time = items <= slots ? most : count == 1 ? rounds * most : std::max(most, all / slots + 0.6 * least);
  return 3 + time + (join > 0 ? 2.5 + join : 0);
}

// A sum of 16-bit products stays in one accumulator, which the tensor cores cut off some 2e-8 of its size after every 16 products: beyond 131072
// products that comes near float16's rounding, so longer sums are split, into 64 at most, whatever the number of tiles.
constexpr int kLongSum = 2048;   // slabs

// The tiles and splits of a launch's products with the least estimated time.
Plan choose_plan(const Sizes* z, int count, int type) {
  Plan best = {1, 0, {{128, 1}, {128, 1}}};
  double best_time = 1e30;
  for (int cg = 1; cg <= 2; cg++) {
    const int slots = kSms / cg;
    std::vector<Config> may[kProblems];
    for (int i = 0; i < count; i++) {
      const long long N = z[i].N, slabs = (z[i].K + kDepth - 1) / kDepth;
      for (int bn = 128 * cg; bn >= 32 * cg; bn -= 16 * cg) {
        const int next = bn - 16 * cg;
        if (bn > 32 * cg && (N + bn - 1) / bn == (N + next - 1) / next) continue;   // a narrower tile covers N as often
        const double tiles = (double)((z[i].M + 128 * cg - 1) / (128 * cg)) * ((N + bn - 1) / bn);
        bool was_long = false;
        static const int kSplits[] = {1, 2, 3, 4, 5, 6, 8, 12, 16, 24, 32, 48, 64};
        for (int splits : kSplits) {
          const bool long_sum = type != GELIB_F32 && slabs > (long long)kLongSum * splits && splits < 64;
          if (splits > 1 && !was_long && (splits > slabs || tiles * splits > 2 * slots || slabs / splits < (type == GELIB_F32 ? 2 : 4))) break;
          was_long = long_sum;
          if (long_sum) continue;
          const long long per = (slabs + splits - 1) / splits;
          may[i].push_back({bn, (int)((slabs + per - 1) / per)});
        }
      }
    }
    for (const Config& c0 : may[0]) {
      Work w[kProblems] = {work_of(z[0], cg, c0, type), {}};
      if (count == 1) {
        const double t = launch_time(w, 1, slots);
        if (t < best_time) best_time = t, best = {cg, 0, {c0, c0}};
        continue;
      }
      for (const Config& c1 : may[1]) {
        w[1] = work_of(z[1], cg, c1, type);
        const double t = launch_time(w, 2, slots);
        if (t < best_time) best_time = t, best = {cg, 0, {c0, c1}};
      }
    }
  }
  if (count == 2) {   // whether handing every other round out backwards evens the blocks' times out
    Work w[kProblems] = {work_of(z[0], best.cg, best.c[0], type), work_of(z[1], best.cg, best.c[1], type)};
    if (w[1].each > w[0].each) std::swap(w[0], w[1]);
    const int slots = kSms / best.cg;
    const double items = w[0].items + w[1].items;
    if (items <= 16.0 * slots) {
      double most[2] = {0, 0};
      for (int flip = 0; flip < 2; flip++) {
        std::vector<double> load(slots, 0.0);
        for (int i = 0; i < (int)items; i++) {
          const int round = i / slots, at = i % slots;
          double& l = load[flip && (round & 1) ? slots - 1 - at : at];
          l += i < w[0].items ? w[0].each : w[1].each;
          most[flip] = std::max(most[flip], l);
        }
      }
      best.flip = most[1] < most[0];
    }
  }
  return best;
}

// Plans are kept by sizes and type: finding one takes some ten microseconds.
Plan plan_of(const Gemm* g, int count) {
  Sizes z[kProblems];
  std::vector<long long> key = {g[0].type};
  for (int i = 0; i < count; i++) {
    z[i] = {g[i].M, g[i].N, g[i].K};
    key.insert(key.end(), {g[i].M, g[i].N, g[i].K});
  }
  static std::mutex mu;
  static std::map<std::vector<long long>, Plan> known;
  {
    std::lock_guard<std::mutex> lock(mu);
    auto it = known.find(key);
    if (it != known.end()) return it->second;
  }
  const Plan plan = choose_plan(z, count, g[0].type);
  std::lock_guard<std::mutex> lock(mu);
  if (known.size() > 4096) known.clear();
  return known[key] = plan;
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
int launch_as(const TcMaps& maps, const TcArgs& a, bool follows, cudaStream_t stream) {
  static const char* fn = "linear";
  auto kernel = gemm_tc_kernel<T, CG, P>;
  constexpr int shared = Shape<CG, P>::kShared;
  static std::atomic<uint64_t> allowed{0};   // devices on which the kernel may have this much shared memory
  int device = 0;
  GELIB_CUDA_TRY(fn, cudaGetDevice(&device));
  const uint64_t bit = device < 64 ? 1ull << device : 0;
  if (!(allowed.load(std::memory_order_relaxed) & bit)) {
    GELIB_CUDA_TRY(fn, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, shared));
    allowed.fetch_or(bit, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t c = {};
  c.gridDim = dim3((unsigned)std::min(a.items, kSms / CG) * CG);
  c.blockDim = dim3(kThreads);
  c.dynamicSmemBytes = shared;
  c.stream = stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = CG, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  c.attrs = CG > 1 ? at : at + 1;
  c.numAttrs = (CG > 1) + follows;
  GELIB_CUDA_TRY(fn, cudaLaunchKernelEx(&c, kernel, maps, a));
  return launched(fn);
}

template <class T, int P>
int launch_config(int cg, const TcMaps& maps, const TcArgs& a, bool follows, cudaStream_t stream) {
  return cg == 2 ? launch_as<T, 2, P>(maps, a, follows, stream) : launch_as<T, 1, P>(maps, a, follows, stream);
}

}  // namespace

bool tc_ready(const Stored& s, int type) {
  if (type == GELIB_F32 && s.planes != 3) return false;
  return is_aligned(s.base, 16) && (s.rows <= 1 || s.ld % 8 == 0);
}

long long tc_gemm_workspace(const Gemm* g, int count) {
  const Plan p = plan_of(g, count);
  long long bytes = 0;
  for (int i = 0; i < count; i++)
    if (p.c[i].splits > 1) bytes += (p.c[i].splits * g[i].M * g[i].N * 4 + 255) / 256 * 256;
  return bytes;
}

int launch_tc_gemm(const Gemm* g, int count, bool follows, void* workspace, Joins* joins, cudaStream_t stream) {
  static const char* fn = "linear";
  const Plan plan = plan_of(g, count);
  TcMaps maps;
  TcArgs a = {};
  char* at = (char*)workspace;
  const Work w0 = work_of({g[0].M, g[0].N, g[0].K}, plan.cg, plan.c[0], g[0].type);
  const bool swapped = count == 2 && work_of({g[1].M, g[1].N, g[1].K}, plan.cg, plan.c[1], g[1].type).each > w0.each;   // longer items first
  for (int i = 0; i < count; i++) {
    const Gemm& q = g[i];
    const Config& c = plan.c[i];
    const int k = swapped ? 1 - i : i;
    // rows across the sum: 64 deep and a tile's rows; rows along it: 64 columns and 64 deep
    if (!encode(&maps.a[k], q.a.s, q.type, 64, q.a.by_sum ? 64 : 128) || !encode(&maps.b[k], q.b.s, q.type, 64, q.b.by_sum ? 64 : c.bn / plan.cg))
      return fail(GELIB_CUDA_ERROR, fn, "a tensor map could not be made");
    TcProblem& p = a.p[k];
    p.e = q.e;
    if (c.splits > 1) {
      p.part = (float*)at;
      at += (c.splits * q.M * q.N * 4 + 255) / 256 * 256;
      joins->add(q, p.part, c.splits);
    }
    p.M = q.M, p.N = (int)q.N;
    p.slabs = (int)((q.K + kDepth - 1) / kDepth);
    p.per = (p.slabs + c.splits - 1) / c.splits;
    p.splits = c.splits;
    const long long tm = (q.M + 128 * plan.cg - 1) / (128 * plan.cg), tn = (q.N + c.bn - 1) / c.bn;
    if (tm * tn * c.splits > 0x1fffffffLL) return fail(GELIB_INVALID, fn, "too many elements");
    p.tiles_m = (int)tm, p.tiles_n = (int)tn, p.items = (int)(tm * tn * c.splits);
    p.bn = c.bn;
    p.a_across = q.a.by_sum, p.b_across = q.b.by_sum;
    const int four = 4 * type_bytes(q.type);
    p.vec = q.N % 4 == 0 && is_aligned(q.e.y, four) && is_aligned(q.e.z, four) && is_aligned(q.e.residual, four);
    a.items += p.items;
  }
  if (count == 1) maps.a[1] = maps.a[0], maps.b[1] = maps.b[0];
  a.flip = plan.flip;
  a.status = async_status_word(kStatusGemmTc);
  a.limit = inject_timeout() ? 0 : kWaitLimit;
  a.bf16 = g[0].type != GELIB_F16;
  if (g[0].type == GELIB_F32) return launch_config<float, 3>(plan.cg, maps, a, follows, stream);
  if (g[0].type == GELIB_BF16) return launch_config<__nv_bfloat16, 1>(plan.cg, maps, a, follows, stream);
  return launch_config<__half, 1>(plan.cg, maps, a, follows, stream);
}

}  // namespace gelib_b200
