// D = A B on the 5th-generation tensor cores: the kernel that gemm_tc.cu (dense layers) and loss_tc.cu (losses and their gradients) give their epilogues.
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
#pragma once
#include <cuda.h>

#include <algorithm>
#include <atomic>

#include "readout.h"
#include "linear.h"
#include "plan.h"
#include "tc_common.h"
#include "tma_maps.h"

namespace gelib_b200 {

constexpr int kProblems = 2;           // of a launch, at most
constexpr int kSms = 148;

// Tiles and splits of a launch's products.
struct Config {
  int bn, splits;
};
struct Plan {
  int cg, flip, lead;
  Config c[kProblems];
};
struct Sizes {
  long long M, N, K;
};
// With `whole` no sum is split.  The longer items of two products go first: `swapped`, whether these are the second's.
Plan plan_of(const Sizes* z, int count, int type, bool whole);
bool swapped(const Plan& plan, const Sizes* z, int count, int type);
bool encode(CUtensorMap* map, const Stored& s, int type, int box_x, int box_y);

namespace {

using tc::smem_u32;

constexpr int kDepth = 64;            // of a slab: 128 bytes of 16-bit numbers
constexpr int kWarps = 8;              // that take the results: two for each quarter of tensor memory, which share a tile's columns
constexpr int kThreads = 96 + 32 * kWarps;   // beside two warps for copies and one for multiplications
constexpr int kChunk = 16;             // columns that such a warp takes at a time, every other chunk of the tile
constexpr int kPitch = kChunk + 4;     // floats of a staged row: 16-byte accesses by rows and by columns without conflicts
constexpr int kStaging = kWarps * 32 * kPitch * 4;

// Where one product of a launch lies; an epilogue's Problem has this as its base.
struct TcShape {
  long long M;
  int N;
  int slabs, per;                     // slabs of the sum, and of one split
  int splits, tiles_m, tiles_n, items;
  int bn;                             // columns of a tile
  int a_across, b_across;             // the operand's rows are the sum's index
};
template <class Problem>
struct TcArgs {
  Problem p[kProblems];               // those with longer items first
  int items;                          // of all
  int flip;                           // every other round of items is handed out from the last block on
  int lead;                           // not 0: so many of the second product's items go to each block that has one of the first's less, before the others get any
  int* status;
  int limit;                          // of the first waits: kWaitLimit, or 0 where a test makes them run out
  int bf16;
  int leave;                          // slabs after which sums leave tensor memory
  const int* other;                   // null, or not zero where maps.other stands for the operand (B if other_b) of problem other_of
  int other_of, other_b;
};
struct TcMaps {
  CUtensorMap a[kProblems], b[kProblems];
  CUtensorMap other;                  // of an operand that there are two of, where args.other says to take it
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
__device__ __forceinline__ Item item_of(const TcShape& g, int i) {
  const int tiles = g.tiles_m * g.tiles_n, t = i % tiles, split = i / tiles;
  // groups of eight tiles of rows, so that the tiles at work at a time share operands in L2
  const int width = 8 * g.tiles_n, first = t / width * 8, high = min(8, g.tiles_m - first);
  return {first + t % width % high, t % width / high, split, split * g.per, min(g.slabs, (split + 1) * g.per)};
}

// The items of a block (or pair) in their order: item `at` of problem `which`, until there are no more.
struct Walk {
  int round, at, which;
  template <class Args>
  __device__ __forceinline__ bool next(const Args& a, int mine, int blocks) {
    const int first = a.p[0].items;
    if (a.lead == 0) {
      at = round * blocks + (a.flip && (round & 1) ? blocks - 1 - mine : mine);
    } else {
      const int whole = first / blocks, more = first - whole * blocks, r = round - whole - (mine < more);   // r: number of the block's item of the second
      if (r < 0) at = round * blocks + mine;
      else if (mine >= more && r < a.lead) at = first + r * (blocks - more) + mine - more;
      else at = first + a.lead * (blocks - more) + (mine >= more ? r - a.lead : r) * blocks + mine;
    }
    round++;
    if (at >= a.items) return false;
    which = at >= first;
    if (which) at -= first;
    return true;
  }
};

constexpr int kAcross = kChunk / 4, kRows = 32 / kAcross, kPasses = 32 / kRows;

// E: what becomes of the sums.  For every item an E is made; `ahead` is told where the item lies (before the first sums are there, or with P = 3 after
// the last), `take` gets the warp's chunks of 16 columns, a row per lane, `has` telling which there are, and `end` comes last.  Before all items the
// epilogue's threads of all blocks may do something else (kBefore).
// kLeave: the sums leave tensor memory after every slab (P = 3) or args.leave of them, and are added in registers, with rounding; otherwise they stay to the end.
template <class E, int CG, int P, bool kLeave>
__global__ void __launch_bounds__(kThreads, 1) gemm_tc_kernel(const __grid_constant__ TcMaps maps, const __grid_constant__ TcArgs<typename E::Problem> args) {
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
    const int other_of = args.other && (args.other_b != 0) == of_b && *args.other ? args.other_of : -1;
    while (ok && walk.next(args, mine_of, blocks)) {
      const TcShape& g = args.p[walk.which];
      const Item it = item_of(g, walk.at);
      const bool across = of_b ? g.b_across : g.a_across;
      const CUtensorMap* map = walk.which == other_of ? &maps.other : of_b ? &maps.b[walk.which] : &maps.a[walk.which];
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
      const TcShape& g = args.p[walk.which];
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
        int next = k0 + args.leave;
        for (int k = k0; k < k1; k++) {
          if constexpr (kLeave)
            if (k == next) {
              end();
              if (!begin()) break;
              next += args.leave;
            }
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
    if constexpr (E::kBefore) E::before(args.p[0], (blockIdx.x * kWarps + warp - 3) * 32 + lane, gridDim.x * kWarps * 32);
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
      const typename E::Problem g = E::kTwo && walk.which ? args.p[1] : args.p[0];   // in registers: the choice costs a load at every use otherwise
      const Item it = item_of(g, walk.at);
      const long long m0 = ((long long)it.m * CG + rank) * 128 + q * 32;
      const int n0 = it.n * g.bn + mine;
      const uint32_t from = tmem + ((uint32_t)q << 21) + mine;
      auto has = [&](int c) { return c < kChunks && mine + c * 2 * kChunk < g.bn && n0 + c * 2 * kChunk < g.N; };
      E e;
      if constexpr (!kLeave) {
        e.template ahead<kChunks>(g, it, m0, n0, lane, mine != 0);
        if (!(ok = all_wait(&bars.sums_full[buf], buf_phase, args.limit))) break;
        tc::tc_fence_after();
#pragma unroll
        for (int c = 0; c < kChunks; c++)
          if (has(c)) {
            uint32_t r[kChunk];
            tc::tmem_ld16(from + buf * S::kBnMost + c * 2 * kChunk, r);
            e.take(g, c, n0 + c * 2 * kChunk, lane, block, r, has(c + 1));
          }
        taken();
      } else {
        if constexpr (P == 1) e.template ahead<kChunks>(g, it, m0, n0, lane, mine != 0);
        float sum[kChunks][kChunk];
#pragma unroll
        for (int c = 0; c < kChunks; c++)
#pragma unroll
          for (int j = 0; j < kChunk; j++) sum[c][j] = 0;
        for (int k = it.k0; k < it.k1; k += P == 3 ? 1 : args.leave) {
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
        if constexpr (P != 1) e.template ahead<kChunks>(g, it, m0, n0, lane, mine != 0);   // no registers for it before
#pragma unroll
        for (int c = 0; c < kChunks; c++)
          if (has(c)) {
            uint32_t r[kChunk];
#pragma unroll
            for (int j = 0; j < kChunk; j++) r[j] = __float_as_uint(sum[c][j]);
            e.take(g, c, n0 + c * 2 * kChunk, lane, block, r, has(c + 1));
          }
      }
      e.end(g, lane);
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

template <class E, int CG, int P, bool kLeave>
int launch_as(const char* fn, const TcMaps& maps, const TcArgs<typename E::Problem>& a, bool follows, cudaStream_t stream) {
  auto kernel = gemm_tc_kernel<E, CG, P, kLeave>;
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

template <class E, int P, bool kLeave = P == 3>
int launch_config(const char* fn, int cg, const TcMaps& maps, const TcArgs<typename E::Problem>& a, bool follows, cudaStream_t stream) {
  return cg == 2 ? launch_as<E, 2, P, kLeave>(fn, maps, a, follows, stream) : launch_as<E, 1, P, kLeave>(fn, maps, a, follows, stream);
}


// The shape of product k of a launch, and its operands' maps; GELIB_OK or an error.
inline int shape_of(const char* fn, const Plan& plan, const Config& c, const Sizes& z, const Operand& a, const Operand& b, int type, TcShape* p, CUtensorMap* map_a,
                    CUtensorMap* map_b) {
  // rows across the sum: 64 deep and a tile's rows; rows along it: 64 columns and 64 deep
  if (!encode(map_a, a.s, type, 64, a.by_sum ? 64 : 128) || !encode(map_b, b.s, type, 64, b.by_sum ? 64 : c.bn / plan.cg))
    return fail(GELIB_CUDA_ERROR, fn, "a tensor map could not be made");
  p->M = z.M, p->N = (int)z.N;
  p->slabs = (int)((z.K + kDepth - 1) / kDepth);
  p->per = (p->slabs + c.splits - 1) / c.splits;
  p->splits = c.splits;
  const long long tm = (z.M + 128 * plan.cg - 1) / (128 * plan.cg), tn = (z.N + c.bn - 1) / c.bn;
  if (tm * tn * c.splits > 0x1fffffffLL) return fail(GELIB_INVALID, fn, "too many elements");
  p->tiles_m = (int)tm, p->tiles_n = (int)tn, p->items = (int)(tm * tn * c.splits);
  p->bn = c.bn;
  p->a_across = a.by_sum, p->b_across = b.by_sum;
  return GELIB_OK;
}
template <class Args>
void finish_args(Args* a, const Plan& plan, int type) {
  a->flip = plan.flip, a->lead = plan.lead;
  a->status = async_status_word(kStatusGemmTc);
  a->limit = inject_timeout() ? 0 : kWaitLimit;
  a->bf16 = type != GELIB_F16;
}

}  // namespace

}  // namespace gelib_b200
