// extern "C" entry points of embedding tables and losses: argument checks, then the kernels.  No exception passes them.
#include <exception>

#include "heads.h"
#include "plan.h"

using namespace gelib_b200;

namespace {

template <class F>
int guarded(const char* fn, F f) {
  try {
    return f();
  } catch (const std::exception& e) {
    return fail(GELIB_INVALID, fn, e.what());
  } catch (...) {
    return fail(GELIB_INVALID, fn, "unknown error");
  }
}

int check_embedding(const char* fn, long long n, int v, int d, int type) {
  if (n < 0 || v < 0 || d < 0) return fail(GELIB_INVALID, fn, "negative size");
  if (n > 1LL << 30 || v > 1 << 30 || d > 1 << 20) return fail(GELIB_INVALID, fn, "more than 2^30 rows, or more than 2^20 columns");
  if (!known_type(type)) return fail(GELIB_INVALID, fn, "unknown type");
  return GELIB_OK;
}

int check_loss(const char* fn, const gelib_linear_loss_args* p, bool back) {
  if (!p) return fail(GELIB_INVALID, fn, "null pointer");
  if (p->m < 0 || p->k < 1 || p->n < 1) return fail(GELIB_INVALID, fn, "negative size, no input channels or no classes");
  if (p->m > 1LL << 30 || p->n > 1 << 30 || p->k > 65536) return fail(GELIB_INVALID, fn, "more than 2^30 rows or classes, or more than 65536 input channels");
  if (!known_type(p->type) || (p->teacher && !known_type(p->teacher_type))) return fail(GELIB_INVALID, fn, "unknown type");
  if (p->index_bytes != 8 && p->index_bytes != 4) return fail(GELIB_INVALID, fn, "numbers of classes have 8 or 4 bytes");
  if (p->reduction < GELIB_LOSS_NONE || p->reduction > GELIB_LOSS_MEAN) return fail(GELIB_INVALID, fn, "unknown reduction");
  if (p->top < 1 || p->top > GELIB_LOSS_MAX_TOP) return fail(GELIB_INVALID, fn, "a row has 1 to GELIB_LOSS_MAX_TOP of the teacher's logits");
  if (p->m && !p->teacher && p->top != 1) return fail(GELIB_INVALID, fn, "several classes per row without a teacher");
  if (p->teacher && !(p->temperature >= 1e-15 && p->temperature <= 1e15)) return fail(GELIB_INVALID, fn, "the temperature is not between 1e-15 and 1e15");
  if (p->ldx < p->k || p->ldw < (p->w_transposed ? p->k : p->n)) return fail(GELIB_INVALID, fn, "rows overlap");
  const int width = type_bytes(p->type);
  for (const void* q : {p->x, p->w, p->bias, (const void*)p->gx, (const void*)p->gw, (const void*)p->gb})
    if (!is_aligned(q, width)) return fail(GELIB_INVALID, fn, "data pointer not aligned to its type");
  if (!is_aligned(p->gy, 4) || !is_aligned(p->loss, 4) || !is_aligned(p->target, p->index_bytes) || (p->teacher && !is_aligned(p->teacher, type_bytes(p->teacher_type))))
    return fail(GELIB_INVALID, fn, "data pointer not aligned to its type");
  if (!is_aligned(p->state, 256)) return fail(GELIB_INVALID, fn, "the state is not 256-byte aligned");
  if (p->m && (!p->x || !p->w || !p->target || !p->state || (back ? !p->gy : !p->loss))) return fail(GELIB_INVALID, fn, "null pointer");
  return GELIB_OK;
}

}  // namespace

extern "C" {

long long gelib_embedding_state_bytes(long long n, int v) { return n > 0 && v > 0 && n <= 1LL << 30 && v <= 1 << 30 ? embedding_state_bytes(n, v) : 0; }

int gelib_embedding(void* y, const void* ids, const void* weight, long long n, int v, int d, long long ldw, double scale, long long padding, int index_bytes,
                    int type, void* state, void* stream) {
  static const char* fn = "embedding";
  return guarded(fn, [&]() -> int {
    const int st = check_embedding(fn, n, v, d, type);
    if (st != GELIB_OK || n == 0) return st;
    if (index_bytes != 8 && index_bytes != 4) return fail(GELIB_INVALID, fn, "numbers of rows have 8 or 4 bytes");
    if (!ids || (d && (!y || (v && !weight)))) return fail(GELIB_INVALID, fn, "null pointer");
    if (ldw < d) return fail(GELIB_INVALID, fn, "rows overlap");
    if (!is_aligned(y, type_bytes(type)) || !is_aligned(weight, type_bytes(type)) || !is_aligned(ids, index_bytes))
      return fail(GELIB_INVALID, fn, "data pointer not aligned to its type");
    if (!is_aligned(state, 256)) return fail(GELIB_INVALID, fn, "the state is not 256-byte aligned");
    return launch_embedding({y, nullptr, ids, weight, nullptr, n, ldw, padding, v, d, index_bytes, type, (float)scale}, v ? state : nullptr, (cudaStream_t)stream);
  });
}

long long gelib_embedding_workspace(long long n, int v, int d, int type) {
  if (n <= 0 || v <= 0 || d <= 0 || n > 1LL << 30 || v > 1 << 30 || d > 1 << 20 || !known_type(type)) return 0;
  return embedding_workspace(n, v, d, type);
}

int gelib_embedding_back(void* gw, const void* gy, const void* state, long long n, int v, int d, double scale, int type, void* workspace, void* stream) {
  static const char* fn = "embedding_back";
  return guarded(fn, [&]() -> int {
    const int st = check_embedding(fn, n, v, d, type);
    if (st != GELIB_OK || v == 0 || d == 0) return st;
    if (!gw || (n && (!gy || !state))) return fail(GELIB_INVALID, fn, "null pointer");
    if (!is_aligned(gw, type_bytes(type)) || !is_aligned(gy, type_bytes(type))) return fail(GELIB_INVALID, fn, "data pointer not aligned to its type");
    if (!is_aligned(workspace, 256) || !is_aligned(state, 256)) return fail(GELIB_INVALID, fn, "the workspace or the state is not 256-byte aligned");
    if (n == 0) {
      GELIB_CUDA_TRY(fn, cudaMemsetAsync(gw, 0, (size_t)v * d * type_bytes(type), (cudaStream_t)stream));
      return GELIB_OK;
    }
    if (!workspace && embedding_workspace(n, v, d, type) > 0) return fail(GELIB_INVALID, fn, "no workspace");
    return launch_embedding_back({nullptr, gw, nullptr, nullptr, gy, n, 0, -1, v, d, 8, type, (float)scale}, state, workspace, (cudaStream_t)stream);
  });
}

long long gelib_linear_loss_state_bytes(const gelib_linear_loss_args* p) {
  return p && p->m >= 0 && p->m <= 1LL << 30 && p->n >= 1 && p->n <= 1 << 30 && p->top >= 1 && p->top <= GELIB_LOSS_MAX_TOP ? linear_loss_state_bytes(*p) : 0;
}

long long gelib_linear_loss_workspace(const gelib_linear_loss_args* p, int backward) {
  long long bytes = 0;
  guarded("linear_loss_workspace", [&]() -> int {
    const int st = check_loss("linear_loss_workspace", p, backward != 0);
    if (st == GELIB_OK && p->m) bytes = linear_loss_workspace(*p, backward != 0);
    return st;
  });
  return bytes;
}

int gelib_linear_loss(const gelib_linear_loss_args* p, void* workspace, void* stream) {
  static const char* fn = "linear_loss";
  return guarded(fn, [&]() -> int {
    int st = poll_async_status(fn);
    if (st == GELIB_OK) st = check_loss(fn, p, false);
    if (st != GELIB_OK) return st;
    if (p->m == 0) {   // the sum of nothing
      if (p->reduction != GELIB_LOSS_NONE && p->loss) GELIB_CUDA_TRY(fn, cudaMemsetAsync(p->loss, 0, 4, (cudaStream_t)stream));
      return GELIB_OK;
    }
    if (!workspace && linear_loss_workspace(*p, false) > 0) return fail(GELIB_INVALID, fn, "no workspace");
    if (!is_aligned(workspace, 256)) return fail(GELIB_INVALID, fn, "the workspace is not 256-byte aligned");
    return launch_linear_loss(*p, workspace, (cudaStream_t)stream);
  });
}

int gelib_linear_loss_back(const gelib_linear_loss_args* p, void* workspace, void* stream) {
  static const char* fn = "linear_loss_back";
  return guarded(fn, [&]() -> int {
    int st = poll_async_status(fn);
    if (st == GELIB_OK) st = check_loss(fn, p, true);
    if (st != GELIB_OK) return st;
    if (p->m == 0) {   // sums of nothing
      const size_t width = type_bytes(p->type);
      if (p->gw) GELIB_CUDA_TRY(fn, cudaMemsetAsync(p->gw, 0, (size_t)p->k * p->n * width, (cudaStream_t)stream));
      if (p->gb) GELIB_CUDA_TRY(fn, cudaMemsetAsync(p->gb, 0, (size_t)p->n * width, (cudaStream_t)stream));
      return GELIB_OK;
    }
    if (!workspace && linear_loss_workspace(*p, true) > 0) return fail(GELIB_INVALID, fn, "no workspace");
    if (!is_aligned(workspace, 256)) return fail(GELIB_INVALID, fn, "the workspace is not 256-byte aligned");
    return launch_linear_loss_back(*p, workspace, (cudaStream_t)stream);
  });
}

}  // extern "C"
