// extern "C" entry points of the readout and the training step: argument checks, then the kernels.  No exception passes them.
#include <algorithm>
#include <cmath>
#include <exception>

#include "readout.h"
#include "linear.h"
#include "norm.h"
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

int check_norm(const char* fn, long long b, long long s, int n, int groups, double eps, int act, int type) {
  if (b < 0 || s < 0 || n < 0 || groups < 1 || n % groups) return fail(GELIB_INVALID, fn, "negative size, or channels that do not divide into the groups");
  if (!known_activation(act) || !known_type(type)) return fail(GELIB_INVALID, fn, "unknown activation or type");
  if (!(eps >= 0)) return fail(GELIB_INVALID, fn, "eps is negative");
  if (n > GELIB_NORM_MAX_CHANNELS) return fail(GELIB_INVALID, fn, "more than GELIB_NORM_MAX_CHANNELS channels");
  if (n && (b > (1LL << 40) / n || s > (1LL << 50) / n / std::max(b, 1LL))) return fail(GELIB_INVALID, fn, "too many elements");
  return GELIB_OK;
}

int check_linear(const char* fn, const gelib_linear_args* p, bool back) {
  if (!p) return fail(GELIB_INVALID, fn, "null pointer");
  if (p->m < 0 || p->k < 0 || p->n < 0) return fail(GELIB_INVALID, fn, "negative size");
  if (!known_activation(p->act) || !known_type(p->type)) return fail(GELIB_INVALID, fn, "unknown activation or type");
  if (p->ldx < p->k || p->ldw < (p->w_transposed ? p->k : p->n)) return fail(GELIB_INVALID, fn, "rows overlap");
  if (p->m > 1LL << 30 || p->k > 1 << 30 || p->n > 1 << 30) return fail(GELIB_INVALID, fn, "more than 2^30 rows or columns");
  const int width = type_bytes(p->type);
  for (const void* q : {p->x, p->w, p->bias, p->residual, p->gy, (const void*)p->y, (const void*)p->z, (const void*)p->gx, (const void*)p->gw, (const void*)p->gb})
    if (!is_aligned(q, width)) return fail(GELIB_INVALID, fn, "data pointer not aligned to its type");
  if (p->m && p->n) {
    if (p->k && (!p->x || !p->w)) return fail(GELIB_INVALID, fn, "null pointer");
    if (back ? !p->gy || (p->act != GELIB_ACT_NONE && !p->z) : !p->y) return fail(GELIB_INVALID, fn, "null pointer");
  }
  return GELIB_OK;
}

bool all_aligned(int bytes, std::initializer_list<const void*> p) {
  for (const void* q : p)
    if (!is_aligned(q, bytes)) return false;
  return true;
}

}  // namespace

extern "C" {

int gelib_adamw_step(int count, const gelib_adamw_tensor* t, const gelib_adamw_options* o, void* stream) {
  static const char* fn = "adamw_step";
  return guarded(fn, [&]() -> int {
    if (count < 0 || (count && !t) || !o) return fail(GELIB_INVALID, fn, "negative count or null pointer");
    if (o->state_bits != 32 && o->state_bits != 8) return fail(GELIB_INVALID, fn, "states have 32 or 8 bits");
    if (o->step < 1) return fail(GELIB_INVALID, fn, "steps are counted from 1");
    if (!(o->beta1 >= 0 && o->beta1 < 1 && o->beta2 >= 0 && o->beta2 < 1)) return fail(GELIB_INVALID, fn, "betas must be in [0, 1)");
    if (!(o->eps >= 0) || !(o->weight_decay >= 0) || !std::isfinite(o->lr)) return fail(GELIB_INVALID, fn, "eps or weight_decay is negative, or lr no number");
    for (int i = 0; i < count; i++) {
      const gelib_adamw_tensor& x = t[i];
      if (x.n < 0 || !known_type(x.type)) return fail(GELIB_INVALID, fn, "negative size or unknown type");
      if (x.n == 0) continue;
      if (!x.p || !x.g || !x.m || !x.v) return fail(GELIB_INVALID, fn, "null pointer");
      if ((x.type == GELIB_F32) != !x.master) return fail(GELIB_INVALID, fn, "a master copy goes with 16-bit parameters, and only with these");
      if (o->state_bits == 8 && (!x.m_scale || !x.v_scale)) return fail(GELIB_INVALID, fn, "8-bit states need their scales");
      const int width = type_bytes(x.type), state = o->state_bits == 8 ? 1 : 4;
      if (!is_aligned(x.p, width) || !is_aligned(x.g, width) || !is_aligned(x.m, state) || !is_aligned(x.v, state) || !is_aligned(x.master, 4) ||
          !is_aligned(x.m_scale, 4) || !is_aligned(x.v_scale, 4))
        return fail(GELIB_INVALID, fn, "data pointer not aligned to its type");
    }
    return launch_adamw(count, t, *o, (cudaStream_t)stream);
  });
}

int gelib_block8_values(void* out, const void* codes, const float* scale, long long n, void* stream) {
  static const char* fn = "block8_values";
  return guarded(fn, [&]() -> int {
    if (n < 0 || (n && (!out || !codes || !scale))) return fail(GELIB_INVALID, fn, "negative size or null pointer");
    if (!is_aligned(out, 2) || !is_aligned(scale, 4)) return fail(GELIB_INVALID, fn, "data pointer not aligned to its type");
    return launch_block8_values(out, codes, scale, n, (cudaStream_t)stream);
  });
}

long long gelib_group_norm_workspace(long long b, long long s, int n, int groups, int type, int backward) {
  if (b <= 0 || s <= 0 || n <= 0 || groups < 1 || n % groups || !known_type(type) || n > GELIB_NORM_MAX_CHANNELS) return 0;
  return group_norm_workspace(b, s, n, groups, type, backward != 0);
}

int gelib_group_norm(void* y, float* mean, float* rstd, const void* x, const void* weight, const void* bias, long long b, long long s, int n,
                     int groups, double eps, int act, int type, void* workspace, void* stream) {
  static const char* fn = "group_norm";
  return guarded(fn, [&]() -> int {
    int st = check_norm(fn, b, s, n, groups, eps, act, type);
    if (st != GELIB_OK) return st;
    if (b == 0 || s == 0 || n == 0) return GELIB_OK;
    if (!x || !y || !mean != !rstd) return fail(GELIB_INVALID, fn, "null pointer");
    if (!workspace && group_norm_workspace(b, s, n, groups, type, false) > 0) return fail(GELIB_INVALID, fn, "no workspace");
    if (!all_aligned(type_bytes(type), {x, y, weight, bias}) || !all_aligned(4, {mean, rstd}) || !is_aligned(workspace, 256))
      return fail(GELIB_INVALID, fn, "data pointer not aligned to its type");
    return launch_group_norm({y, mean, rstd, x, weight, bias, nullptr, nullptr, nullptr, b, s, n, groups, (float)eps, act, type, (float*)workspace},
                             (cudaStream_t)stream);
  });
}

int gelib_group_norm_back(void* gx, void* gw, void* gb, const void* gy, const void* x, const void* weight, const void* bias, const float* mean,
                          const float* rstd, long long b, long long s, int n, int groups, int act, int type, void* workspace, void* stream) {
  static const char* fn = "group_norm_back";
  return guarded(fn, [&]() -> int {
    int st = check_norm(fn, b, s, n, groups, 0, act, type);
    if (st != GELIB_OK) return st;
    if (n == 0 || (!gx && !gw && !gb)) return GELIB_OK;
    if (b == 0 || s == 0) {  // sums of nothing
      for (void* g : {gw, gb})
        if (g) GELIB_CUDA_TRY(fn, cudaMemsetAsync(g, 0, (size_t)n * type_bytes(type), (cudaStream_t)stream));
      return GELIB_OK;
    }
    if (!x || !gy || !mean || !rstd) return fail(GELIB_INVALID, fn, "null pointer");
    if (!workspace && group_norm_workspace(b, s, n, groups, type, true) > 0) return fail(GELIB_INVALID, fn, "no workspace");
    if (!all_aligned(type_bytes(type), {x, gy, gx, gw, gb, weight, bias}) || !all_aligned(4, {mean, rstd}) || !is_aligned(workspace, 256))
      return fail(GELIB_INVALID, fn, "data pointer not aligned to its type");
    return launch_group_norm({gx, (float*)mean, (float*)rstd, x, weight, bias, gy, gw, gb, b, s, n, groups, 0.f, act, type, (float*)workspace},
                             (cudaStream_t)stream);
  });
}

long long gelib_linear_workspace(const gelib_linear_args* p, int backward) {
  long long bytes = 0;
  guarded("linear_workspace", [&]() -> int {
    const int st = check_linear("linear_workspace", p, backward != 0);
    if (st == GELIB_OK) bytes = linear_workspace(*p, backward != 0);
    return st;
  });
  return bytes;
}

int gelib_linear(const gelib_linear_args* p, void* workspace, void* stream) {
  static const char* fn = "linear";
  return guarded(fn, [&]() -> int {
    int st = poll_async_status(fn);
    if (st == GELIB_OK) st = check_linear(fn, p, false);
    if (st != GELIB_OK || p->m == 0 || p->n == 0) return st;
    if (!workspace && linear_workspace(*p, false) > 0) return fail(GELIB_INVALID, fn, "no workspace");
    if (!is_aligned(workspace, 256)) return fail(GELIB_INVALID, fn, "the workspace is not 256-byte aligned");
    return launch_linear(*p, workspace, (cudaStream_t)stream);
  });
}

int gelib_linear_back(const gelib_linear_args* p, void* workspace, void* stream) {
  static const char* fn = "linear_back";
  return guarded(fn, [&]() -> int {
    int st = poll_async_status(fn);
    if (st == GELIB_OK) st = check_linear(fn, p, true);
    if (st != GELIB_OK) return st;
    if (!workspace && linear_workspace(*p, true) > 0) return fail(GELIB_INVALID, fn, "no workspace");
    if (!is_aligned(workspace, 256)) return fail(GELIB_INVALID, fn, "the workspace is not 256-byte aligned");
    return launch_linear_back(*p, workspace, (cudaStream_t)stream);
  });
}

}  // extern "C"
