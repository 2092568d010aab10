// Dense layers' products: the epilogue of the kernel in gemm_tc.cuh, and the choice of tiles and splits.
#include <cmath>
#include <map>
#include <mutex>
#include <vector>

#include "gemm_tc.cuh"

namespace gelib_b200 {

namespace {

struct TcProblem : TcShape {
  Epilogue e;
  float* part;                        // partial sums (splits, M, N), or null
  int vec;                            // columns may be taken four at a time
};

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

template <class T, int P>
struct DenseEnd {
  using Problem = TcProblem;
  static constexpr bool kTwo = true, kBefore = false;
  Rest<T> rest[2];                    // of a chunk, and of the next, asked for before the first is stored
  float bias[P == 1 ? 8 : 1][4];
  long long m0;
  int split;

  template <int kChunks>
  __device__ __forceinline__ void ahead(const Problem& g, const Item& it, long long m, int n0, int lane, bool) {
    m0 = m, split = it.split;
    if constexpr (P == 1)
#pragma unroll
      for (int c = 0; c < kChunks; c++) load_bias<T>(g, n0 + c * 2 * kChunk, lane, bias[c]);
    load_rest<T>(g, m0, n0, lane, rest[0]);
  }
  __device__ __forceinline__ void take(const Problem& g, int c, int n, int lane, uint32_t block, const uint32_t (&r)[kChunk], bool more) {
    if (more) load_rest<T>(g, m0, n + 2 * kChunk, lane, rest[(c + 1) & 1]);
    if constexpr (P != 1) load_bias<T>(g, n, lane, bias[0]);
    store_chunk<T>(g, split, r, block, m0, n, lane, bias[P == 1 ? c : 0], rest[c & 1]);
  }
  __device__ __forceinline__ void end(const Problem&, int) {}
};

// ---- host -----------------------------------------------------------------------------------------------------------------------------

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
Plan choose_plan(const Sizes* z, int count, int type, bool whole) {
  Plan best = {1, 0, 0, {{128, 1}, {128, 1}}};
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
          if (whole && splits > 1) break;
          const bool long_sum = !whole && type != GELIB_F32 && slabs > (long long)kLongSum * splits && splits < 64;
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
        if (t < best_time) best_time = t, best = {cg, 0, 0, {c0, c0}};
        continue;
      }
      for (const Config& c1 : may[1]) {
        w[1] = work_of(z[1], cg, c1, type);
        const double t = launch_time(w, 2, slots);
        if (t < best_time) best_time = t, best = {cg, 0, 0, {c0, c1}};
      }
    }
  }
  if (count == 2) {   // the way of handing items out that evens the blocks' times out: as they come, every other round backwards, or the longer ones' last round first
    Work w[kProblems] = {work_of(z[0], best.cg, best.c[0], type), work_of(z[1], best.cg, best.c[1], type)};
    if (w[1].each > w[0].each) std::swap(w[0], w[1]);
    const int slots = kSms / best.cg, longer = (int)w[0].items % slots;
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
      best_time = std::min(most[0], most[1]);
    } else {
      best_time = std::ceil(w[0].items / slots) * w[0].each + std::ceil((items - slots * std::ceil(w[0].items / slots)) / slots) * w[1].each;
    }
    const double whole = std::floor(w[0].items / slots);
    if (longer > 0)
      for (int lead = 1; lead <= 2 * w[0].each / w[1].each + 1; lead++) {
        const double rest = std::max(0.0, w[1].items - (double)lead * (slots - longer));
        const double time = whole * w[0].each + std::max(w[0].each, lead * w[1].each) + std::ceil(rest / slots) * w[1].each;
        if (time < 0.97 * best_time) best.flip = 0, best.lead = lead, best_time = time;
      }
  }
  return best;
}

}  // namespace

// Plans are kept by sizes and type: finding one takes some ten microseconds.
Plan plan_of(const Sizes* z, int count, int type, bool whole) {
  std::vector<long long> key = {type, whole};
  for (int i = 0; i < count; i++) key.insert(key.end(), {z[i].M, z[i].N, z[i].K});
  static std::mutex mu;
  static std::map<std::vector<long long>, Plan> known;
  {
    std::lock_guard<std::mutex> lock(mu);
    auto it = known.find(key);
    if (it != known.end()) return it->second;
  }
  const Plan plan = choose_plan(z, count, type, whole);
  std::lock_guard<std::mutex> lock(mu);
  if (known.size() > 4096) known.clear();
  return known[key] = plan;
}

bool swapped(const Plan& plan, const Sizes* z, int count, int type) {
  return count == 2 && work_of(z[1], plan.cg, plan.c[1], type).each > work_of(z[0], plan.cg, plan.c[0], type).each;
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

bool tc_ready(const Stored& s, int type) {
  if (type == GELIB_F32 && s.planes != 3) return false;
  return is_aligned(s.base, 16) && (s.rows <= 1 || s.ld % 8 == 0);
}

namespace {

Plan plan_for(const Gemm* g, int count, Sizes (&z)[kProblems]) {
  for (int i = 0; i < count; i++) z[i] = {g[i].M, g[i].N, g[i].K};
  return plan_of(z, count, g[0].type, false);
}

}  // namespace

long long tc_gemm_workspace(const Gemm* g, int count) {
  Sizes z[kProblems];
  const Plan p = plan_for(g, count, z);
  long long bytes = 0;
  for (int i = 0; i < count; i++)
    if (p.c[i].splits > 1) bytes += (p.c[i].splits * g[i].M * g[i].N * 4 + 255) / 256 * 256;
  return bytes;
}

int launch_tc_gemm(const Gemm* g, int count, bool follows, void* workspace, Joins* joins, cudaStream_t stream) {
  static const char* fn = "linear";
  Sizes z[kProblems];
  const int type = g[0].type;
  const Plan plan = plan_for(g, count, z);
  TcMaps maps = {};
  TcArgs<TcProblem> a = {};
  char* at = (char*)workspace;
  const bool other = swapped(plan, z, count, type);
  for (int i = 0; i < count; i++) {
    const Gemm& q = g[i];
    const Config& c = plan.c[i];
    const int k = other ? 1 - i : i;
    TcProblem& p = a.p[k];
    const int st = shape_of(fn, plan, c, z[i], q.a, q.b, type, &p, &maps.a[k], &maps.b[k]);
    if (st != GELIB_OK) return st;
    p.e = q.e;
    if (c.splits > 1) {
      p.part = (float*)at;
      at += (c.splits * q.M * q.N * 4 + 255) / 256 * 256;
      joins->add(q, p.part, c.splits);
    }
    const int four = 4 * type_bytes(type);
    p.vec = q.N % 4 == 0 && is_aligned(q.e.y, four) && is_aligned(q.e.z, four) && is_aligned(q.e.residual, four);
    a.items += p.items;
  }
  if (count == 1) maps.a[1] = maps.a[0], maps.b[1] = maps.b[0];
  finish_args(&a, plan, type);
  if (type == GELIB_F32) return launch_config<DenseEnd<float, 3>, 3>(fn, plan.cg, maps, a, follows, stream);
  if (type == GELIB_BF16) return launch_config<DenseEnd<__nv_bfloat16, 1>, 1>(fn, plan.cg, maps, a, follows, stream);
  return launch_config<DenseEnd<__half, 1>, 1>(fn, plan.cg, maps, a, follows, stream);
}

}  // namespace gelib_b200
