// extern "C" entry points of the readout and the training step: argument checks, then the kernels.  No exception passes them.
#include <cmath>
#include <exception>

#include "plan.h"
#include "readout.h"

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

}  // extern "C"
