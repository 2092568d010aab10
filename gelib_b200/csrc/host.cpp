// The host side of the Python products, in native code: what SO3part.py, SO3vec.py, readout.py, heads.py and adamw.py do around one C-ABI call --
// output type, output tensors, zero-filled gradients, descriptors, device, stream -- for operands that need nothing special.  Each
// function returns None, having done nothing, when an operand is not plain (not on a CUDA device, not complex64, lazily
// conjugated, more than two grid dimensions, two parts of one l, ...), when sizes do not fit together, and when the library
// skips the call: the Python code then takes it from the start and says what there is to say.
#include <ATen/ATen.h>
#include <ATen/ops/_foreach_zero.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <climits>
#include <optional>
#include <stdexcept>
#include <string>
#include <vector>

#include "../../include/gelib_b200.h"

namespace {

using Tensors = std::vector<at::Tensor>;

// A plain Python int of 32 bits.  Others are left to the Python code too: through ctypes the low 32 bits of a larger maxl count
// (sys.maxsize: every l), and what is not an int is refused there.
std::optional<int> plain_int(pybind11::handle h) {
  if (!PyLong_CheckExact(h.ptr())) return std::nullopt;
  int overflow = 0;
  const long v = PyLong_AsLongAndOverflow(h.ptr(), &overflow);
  if (overflow || v < INT_MIN || v > INT_MAX) return std::nullopt;
  return static_cast<int>(v);
}

// The tensor in canonical form, core/Gpart.hpp:450-469 of GElib; false when it is not plain.
bool describe(const at::Tensor& t, c10::Device device, gelib_tensor5* d) {
  if (!t.defined() || !t.is_cuda() || t.device() != device || t.scalar_type() != at::kComplexFloat || t.is_conj()) return false;
  const int dim = static_cast<int>(t.dim());
  if (dim < 3 || dim > 5) return false;
  const auto sizes = t.sizes();
  const auto strides = t.strides();
  for (int k = 0; k < dim; k++)
    if (sizes[k] > INT_MAX) return false;
  d->base = static_cast<float*>(t.data_ptr());
  const int at[5] = {0, dim > 3 ? 1 : -1, dim > 4 ? 2 : -1, dim - 2, dim - 1};
  for (int k = 0; k < 5; k++) {
    d->dims[k] = at[k] < 0 ? 1 : static_cast<int32_t>(sizes[at[k]]);
    d->strides[k] = at[k] < 0 ? 0 : 2 * strides[at[k]];  // in floats
  }
  return true;
}

// The parts of a vector, described in ascending l.
struct Vec {
  std::vector<gelib_tensor5> d;
  std::vector<int> l, n;
  int size() const { return static_cast<int>(d.size()); }
};
bool describe_all(const Tensors& parts, c10::Device device, Vec* v) {
  std::vector<std::pair<int, const at::Tensor*>> order;
  order.reserve(parts.size());
  for (const auto& t : parts) {
    if (!t.defined() || t.dim() < 3 || t.size(-2) > INT_MAX) return false;
    order.emplace_back(static_cast<int>((t.size(-2) - 1) / 2), &t);
  }
  std::sort(order.begin(), order.end(), [](const auto& a, const auto& b) { return a.first < b.first; });
  for (size_t i = 0; i < order.size(); i++) {
    if (i > 0 && order[i].first == order[i - 1].first) return false;
    gelib_tensor5 t;
    if (!describe(*order[i].second, device, &t)) return false;
    v->d.push_back(t);
    v->l.push_back(order[i].first);
    v->n.push_back(t.dims[4]);
  }
  return true;
}

// Makes the call without the interpreter lock (a first call of a signature builds its plan; autograd's threads do not hold it).  True: done; false: the library
// skipped it.  Errors raise, as in _lib.check.
template <class F>
bool call(F f) {
  int status;
  std::string message;
  {
    std::optional<pybind11::gil_scoped_release> release;
    if (PyGILState_Check()) release.emplace();
    status = f();
    if (status != GELIB_OK && status != GELIB_SKIPPED) message = gelib_last_error();
  }
  if (!message.empty()) throw std::runtime_error(message);
  return status == GELIB_OK;
}

void* stream_of(c10::Device device) { return c10::cuda::getCurrentCUDAStream(device.index()).stream(); }

// Batch and grid of a product; false when the batches do not fit, or an operand is empty (the kernels then write nothing).
bool lead_dims(const at::Tensor& x, const at::Tensor& y, std::vector<int64_t>* lead) {
  const int64_t bx = x.size(0), by = y.size(0);
  if ((bx > 1 && by > 1 && bx != by) || x.numel() == 0 || y.numel() == 0) return false;
  lead->push_back(std::max(bx, by));
  const int64_t gx = x.dim() - 3, gy = y.dim() - 3;
  for (int64_t k = 1; k <= std::max(gx, gy); k++)  // size-1 grid dimensions are broadcast against the other operand's
    lead->push_back(gx == gy ? std::max(x.size(k), y.size(k)) : (gx > gy ? x : y).size(k));
  return true;
}

at::Tensor output(std::vector<int64_t> lead, int64_t l, int64_t n, c10::Device device) {
  lead.push_back(2 * l + 1);
  lead.push_back(n);
  return at::empty(lead, at::TensorOptions().dtype(at::kComplexFloat).device(device));
}

Tensors zeros_like_all(const Tensors& v) {
  Tensors r;
  r.reserve(v.size());
  for (const auto& t : v) r.push_back(at::empty_like(t));
  at::_foreach_zero_(r);
  return r;
}

std::optional<Tensors> vec_forward(const Tensors& x, const Tensors& y, pybind11::handle max_l, bool diag) {
  const auto maxl = plain_int(max_l);
  if (!maxl || x.empty() || y.empty() || !x[0].defined() || !x[0].is_cuda()) return std::nullopt;
  const auto device = x[0].device();
  Vec dx, dy, dr;
  std::vector<int64_t> lead;
  if (!describe_all(x, device, &dx) || !describe_all(y, device, &dy) || !lead_dims(x[0], y[0], &lead)) return std::nullopt;
  const int cap = dx.l.back() + dy.l.back() + 1;
  std::vector<int> l(cap), n(cap);
  const int k = gelib_SO3type_CGproduct(dx.size(), dx.l.data(), dx.n.data(), dy.size(), dy.l.data(), dy.n.data(), *maxl, diag, cap, l.data(), n.data());
  if (k <= 0) return std::nullopt;
  c10::cuda::CUDAGuard guard(device);
  Tensors r;
  for (int i = 0; i < k; i++) r.push_back(output(lead, l[i], n[i], device));
  if (!describe_all(r, device, &dr)) return std::nullopt;
  void* s = stream_of(device);
  const auto f = diag ? gelib_SO3vec_addDiagCGproduct : gelib_SO3vec_addCGproduct;
  if (!call([&] { return f(dr.size(), dr.d.data(), dx.size(), dx.d.data(), dy.size(), dy.d.data(), GELIB_OVERWRITE, s); })) return std::nullopt;
  return r;
}

// The gradients asked for, those of x first.
std::optional<Tensors> vec_backward(const Tensors& x, const Tensors& y, const Tensors& g, bool need_x, bool need_y, bool diag) {
  if (x.empty() || y.empty() || g.empty() || !(need_x || need_y) || !x[0].defined() || !x[0].is_cuda()) return std::nullopt;
  const auto device = x[0].device();
  Vec dx, dy, dg, dxg, dyg;
  if (!describe_all(x, device, &dx) || !describe_all(y, device, &dy) || !describe_all(g, device, &dg)) return std::nullopt;
  Tensors wanted;
  if (need_x) wanted.insert(wanted.end(), x.begin(), x.end());
  if (need_y) wanted.insert(wanted.end(), y.begin(), y.end());
  c10::cuda::CUDAGuard guard(device);
  Tensors r = zeros_like_all(wanted);
  const auto split = r.begin() + (need_x ? x.size() : 0);
  if (!describe_all(Tensors(r.begin(), split), device, &dxg) || !describe_all(Tensors(split, r.end()), device, &dyg)) return std::nullopt;
  void* s = stream_of(device);
  const bool ok = call([&] {
    if (need_x && need_y)
      return (diag ? gelib_SO3vec_addDiagCGproduct_back01 : gelib_SO3vec_addCGproduct_back01)(
          dxg.size(), dxg.d.data(), dyg.size(), dyg.d.data(), dg.size(), dg.d.data(), dx.d.data(), dy.d.data(), 0, s);
    if (need_x)
      return (diag ? gelib_SO3vec_addDiagCGproduct_back0 : gelib_SO3vec_addCGproduct_back0)(dxg.size(), dxg.d.data(), dg.size(), dg.d.data(),
                                                                                           dy.size(), dy.d.data(), 0, s);
    return (diag ? gelib_SO3vec_addDiagCGproduct_back1 : gelib_SO3vec_addCGproduct_back1)(dyg.size(), dyg.d.data(), dg.size(), dg.d.data(),
                                                                                         dx.size(), dx.d.data(), 0, s);
  });
  if (!ok) return std::nullopt;
  return r;
}

std::optional<at::Tensor> part_forward(const at::Tensor& x, const at::Tensor& y, pybind11::handle out_l, bool diag) {
  const auto l = plain_int(out_l);
  if (!l || !x.defined() || !x.is_cuda() || *l < 0) return std::nullopt;
  const auto device = x.device();
  gelib_tensor5 dx, dy, dr;
  std::vector<int64_t> lead;
  if (!describe(x, device, &dx) || !describe(y, device, &dy) || !lead_dims(x, y, &lead)) return std::nullopt;
  if (diag && x.size(-1) != y.size(-1)) return std::nullopt;
  c10::cuda::CUDAGuard guard(device);
  at::Tensor r = output(lead, *l, diag ? x.size(-1) : x.size(-1) * y.size(-1), device);
  if (!describe(r, device, &dr)) return std::nullopt;
  void* s = stream_of(device);
  const auto f = diag ? gelib_SO3part_addDiagCGproduct : gelib_SO3part_addCGproduct;
  if (!call([&] { return f(&dr, &dx, &dy, 0, GELIB_OVERWRITE, s); })) return std::nullopt;
  return r;
}

std::optional<Tensors> part_backward(const at::Tensor& x, const at::Tensor& y, const at::Tensor& g, bool need_x, bool need_y, bool diag) {
  if (!x.defined() || !x.is_cuda() || !(need_x || need_y)) return std::nullopt;
  const auto device = x.device();
  gelib_tensor5 dx, dy, dg, dw[2];
  if (!describe(x, device, &dx) || !describe(y, device, &dy) || !describe(g, device, &dg)) return std::nullopt;
  Tensors wanted;
  if (need_x) wanted.push_back(x);
  if (need_y) wanted.push_back(y);
  c10::cuda::CUDAGuard guard(device);
  Tensors r = zeros_like_all(wanted);
  for (size_t i = 0; i < r.size(); i++)
    if (!describe(r[i], device, &dw[i])) return std::nullopt;
  void* s = stream_of(device);
  const bool ok = call([&] {
    if (need_x && need_y) return (diag ? gelib_SO3part_addDiagCGproduct_back01 : gelib_SO3part_addCGproduct_back01)(&dw[0], &dw[1], &dg, &dx, &dy, 0, 0, s);
    if (need_x) return (diag ? gelib_SO3part_addDiagCGproduct_back0 : gelib_SO3part_addCGproduct_back0)(&dw[0], &dg, &dy, 0, 0, s);
    return (diag ? gelib_SO3part_addDiagCGproduct_back1 : gelib_SO3part_addCGproduct_back1)(&dw[0], &dg, &dx, 0, 0, s);
  });
  if (!ok) return std::nullopt;
  return r;
}

// x gathered along array dimension d (tensor dimension d + 1) by a map of n_in cells into n_out.
std::optional<at::Tensor> gather(const at::Tensor& x0, const at::Tensor& row_ptr, const at::Tensor& col, int n_in, int n_out, pybind11::handle dim) {
  const auto array_dim = plain_int(dim);
  if (!array_dim || !x0.defined() || !x0.is_cuda() || x0.scalar_type() != at::kComplexFloat || x0.is_conj()) return std::nullopt;
  const auto device = x0.device();
  const int d = *array_dim;
  if (d < 0 || d + 1 >= x0.dim() || x0.size(d + 1) != n_in || row_ptr.device() != device || col.device() != device) return std::nullopt;
  c10::cuda::CUDAGuard guard(device);
  const at::Tensor x = x0.detach().contiguous();
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
  shape[d + 1] = n_out;
  int64_t outer = 1, inner = 1;
  for (int k = 0; k <= d; k++) outer *= shape[k];
  for (size_t k = d + 2; k < shape.size(); k++) inner *= shape[k];
  at::Tensor r = at::zeros(shape, at::TensorOptions().dtype(at::kComplexFloat).device(device));
  void* s = stream_of(device);
  float* rp = static_cast<float*>(r.data_ptr());
  const float* xp = static_cast<const float*>(x.data_ptr());
  const int *pp = row_ptr.data_ptr<int>(), *cp = col.data_ptr<int>();
  if (!call([&] { return gelib_add_gather(rp, xp, outer, n_out, n_in, inner, pp, cp, s); })) return std::nullopt;
  return r;
}

using OptTensors = std::vector<std::optional<at::Tensor>>;

std::optional<int> type_code(at::ScalarType t) {
  if (t == at::kFloat || t == at::kComplexFloat) return GELIB_F32;
  if (t == at::kBFloat16) return GELIB_BF16;
  if (t == at::kHalf) return GELIB_F16;
  return std::nullopt;
}

bool plain_dense(const at::Tensor& t, c10::Device device) {
  return t.defined() && t.device() == device && t.layout() == at::kStrided && t.is_contiguous() && !t.is_conj() && !t.is_neg();
}

int64_t reals(const at::Tensor& t) { return t.numel() * (t.is_complex() ? 2 : 1); }

// One step over lists of tensors; None when one of them is not plain, or does not go with the others.
std::optional<bool> adamw_step(const Tensors& params, const Tensors& grads, const Tensors& m, const Tensors& v, const std::optional<Tensors>& ms,
                               const std::optional<Tensors>& vs, const std::optional<OptTensors>& master, int64_t step, double lr, double beta1, double beta2, double eps,
                               double weight_decay, uint64_t seed, const std::optional<at::Tensor>& grad_scale, bool refresh_master) {
  const size_t k = params.size();
  if (k == 0 || grads.size() != k || m.size() != k || v.size() != k || ms.has_value() != vs.has_value()) return std::nullopt;
  if ((ms && (ms->size() != k || vs->size() != k)) || (master && master->size() != k) || !params[0].defined() || !params[0].is_cuda()) return std::nullopt;
  const auto device = params[0].device();
  gelib_adamw_options o = {lr, beta1, beta2, eps, weight_decay, step, seed, nullptr, ms ? 8 : 32, refresh_master};
  if (grad_scale) {
    if (!plain_dense(*grad_scale, device) || grad_scale->scalar_type() != at::kFloat || grad_scale->numel() != 1) return std::nullopt;
    o.grad_scale = grad_scale->data_ptr<float>();
  }
  std::vector<gelib_adamw_tensor> t(k);
  for (size_t i = 0; i < k; i++) {
    const at::Tensor &p = params[i], &g = grads[i];
    if (!plain_dense(p, device) || !plain_dense(g, device) || g.scalar_type() != p.scalar_type() || g.sizes() != p.sizes()) return std::nullopt;
    const auto type = type_code(p.scalar_type());
    if (!type) return std::nullopt;
    const int64_t n = reals(p);
    const auto state = [&](const at::Tensor& s) {
      return plain_dense(s, device) && reals(s) == n && (ms ? s.scalar_type() == at::kFloat8_e4m3fn : s.scalar_type() == at::kFloat || s.scalar_type() == at::kComplexFloat);
    };
    if (!state(m[i]) || !state(v[i])) return std::nullopt;
    t[i] = {p.data_ptr(), nullptr, g.data_ptr(), m[i].data_ptr(), v[i].data_ptr(), nullptr, nullptr, n, *type};
    if (ms) {
      for (const auto* s : {&(*ms)[i], &(*vs)[i]})
        if (!plain_dense(*s, device) || s->scalar_type() != at::kFloat || s->numel() != (n + 255) / 256) return std::nullopt;
      t[i].m_scale = (*ms)[i].data_ptr<float>();
      t[i].v_scale = (*vs)[i].data_ptr<float>();
    }
    const bool has = master && (*master)[i].has_value();
    if (has != (*type != GELIB_F32)) return std::nullopt;
    if (has) {
      const at::Tensor& w = *(*master)[i];
      if (!plain_dense(w, device) || w.scalar_type() != at::kFloat || w.numel() != n) return std::nullopt;
      t[i].master = w.data_ptr<float>();
    }
  }
  c10::cuda::CUDAGuard guard(device);
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) return std::nullopt;
  void* s = stream_of(device);
  call([&] { return gelib_adamw_step(static_cast<int>(k), t.data(), &o, s); });
  // what autograd has saved of these tensors is no longer what they hold
  const auto written = [](const at::Tensor& w) {
    if (!w.is_inference()) w.unsafeGetTensorImpl()->bump_version();
  };
  for (const Tensors* list : {&params, &m, &v, ms ? &*ms : nullptr, vs ? &*vs : nullptr})
    if (list)
      for (const auto& w : *list) written(w);
  if (master)
    for (const auto& w : *master)
      if (w) written(*w);
  return true;
}

std::optional<at::Tensor> block8_values(const at::Tensor& codes, const at::Tensor& scale) {
  if (!codes.defined() || !codes.is_cuda()) return std::nullopt;
  const auto device = codes.device();
  if (!plain_dense(codes, device) || codes.scalar_type() != at::kFloat8_e4m3fn || !plain_dense(scale, device) || scale.scalar_type() != at::kFloat ||
      scale.numel() != (codes.numel() + 255) / 256)
    return std::nullopt;
  c10::cuda::CUDAGuard guard(device);
  at::Tensor out = at::empty(codes.sizes(), at::TensorOptions().dtype(at::kBFloat16).device(device));
  void* s = stream_of(device);
  call([&] { return gelib_block8_values(out.data_ptr(), codes.data_ptr(), scale.data_ptr<float>(), codes.numel(), s); });
  return out;
}

// ---- readout ---------------------------------------------------------------------------------------------------------------------

using OptTensor = std::optional<at::Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void* ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
at::Tensor or_none(const OptTensor& t) { return t ? *t : at::Tensor(); }

// A forward-mode derivative, which these operators do not have: the Python code refuses it.  Asked of every operand, since a tensor with a
// tangent need not ask for a gradient and would lose it here.
bool has_tangent(const at::Tensor& t) { return t._fw_grad(/*level=*/0).defined(); }

// Real, of x's type and device, of the given shape.
bool goes_with(const at::Tensor& x, const OptTensor& t, at::IntArrayRef shape) {
  return !t || (t->defined() && t->device() == x.device() && t->scalar_type() == x.scalar_type() && t->layout() == at::kStrided && t->sizes() == shape && !t->is_neg() &&
                !has_tangent(*t));
}
bool is_plain(const at::Tensor& x) {
  return x.defined() && x.is_cuda() && x.layout() == at::kStrided && !x.is_neg() && !x.is_complex() && type_code(x.scalar_type()).has_value() && !has_tangent(x);
}

at::Tensor workspace(int64_t bytes, const at::Tensor& like) {
  return bytes > 0 ? at::empty({bytes}, like.options().dtype(at::kByte)) : at::Tensor();
}

// Gradients of a call whose own gradient is asked for: an error when that is wanted, not zeros.
variable_list differentiable_once(variable_list grads, const char* name) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list some;
  for (auto& g : grads)
    if (g.defined()) some.push_back(g.detach().requires_grad_());
  auto error = std::make_shared<torch::autograd::DelayedError>(std::string(name) + " can be differentiated once", static_cast<int>(some.size()));
  some = (*error)(std::move(some));
  size_t i = 0;
  for (auto& g : grads)
    if (g.defined()) g = some[i++];
  return grads;
}

// x as rows of n elements `ld` apart, over all its leading dimensions; copied where it does not lie like that.
at::Tensor as_rows(const at::Tensor& x, int64_t n, int64_t* ld) {
  *ld = n;
  if (x.is_contiguous()) return x;
  if (x.dim() == 2 && (x.stride(1) == 1 || n == 1) && x.stride(0) >= n) {
    *ld = x.stride(0);
    return x;
  }
  return x.contiguous();
}

struct Layer {
  gelib_linear_args a = {};
  at::Tensor x, w, z;
};
void describe_layer(Layer* l, const at::Tensor& x, const at::Tensor& w, int act) {
  l->a.k = static_cast<int>(w.size(0));
  l->a.n = static_cast<int>(w.size(1));
  int64_t m = 1;
  for (int64_t d = 0; d + 1 < x.dim(); d++) m *= x.size(d);
  l->a.m = m;
  l->x = as_rows(x, l->a.k, &l->a.ldx);
  // the view v.t() of a matrix (n_out, n_in) is used as it lies
  l->a.w_transposed = w.stride(0) == 1 && w.stride(1) != 1 && w.stride(1) >= l->a.k;
  if (l->a.w_transposed) l->w = w, l->a.ldw = w.stride(1);
  else l->w = as_rows(w, l->a.n, &l->a.ldw);
  l->a.x = l->x.data_ptr(), l->a.w = l->w.data_ptr();
  l->a.act = act, l->a.type = *type_code(x.scalar_type());
}

at::Tensor linear_call(Layer* l, const at::Tensor& x, const at::Tensor& w, const at::Tensor& bias, const at::Tensor& residual, int act, bool keep) {
  c10::cuda::CUDAGuard guard(x.device());
  describe_layer(l, x, w, act);
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = l->a.n;
  const at::Tensor y = at::empty(shape, x.options()), b = bias.defined() ? bias.contiguous() : bias, r = residual.defined() ? residual.contiguous() : residual;
  if (keep && act != GELIB_ACT_NONE) l->z = at::empty({l->a.m, l->a.n}, x.options());
  l->a.bias = ptr(b), l->a.residual = ptr(r), l->a.y = ptr(y), l->a.z = ptr(l->z);
  const at::Tensor space = workspace(gelib_linear_workspace(&l->a, 0), x);
  void* s = stream_of(x.device());
  call([&] { return gelib_linear(&l->a, ptr(space), s); });
  return y;
}

struct LinearFunction : torch::autograd::Function<LinearFunction> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w, const OptTensor& bias, const OptTensor& residual, int64_t act) {
    Layer l;
    const bool keep = x.requires_grad() || w.requires_grad() || (bias && bias->requires_grad());
    at::Tensor y = linear_call(&l, x, w, or_none(bias), or_none(residual), static_cast<int>(act), keep);
    if (keep) ctx->save_for_backward({x, w, l.z});
    ctx->saved_data["act"] = act;
    ctx->saved_data["bias"] = bias.has_value();
    ctx->saved_data["residual"] = residual.has_value();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(5);
    // edges are counted over the tensors that were given
    const bool has_bias = ctx->saved_data["bias"].toBool();
    const bool need[3] = {ctx->needs_input_grad(0), ctx->needs_input_grad(1), has_bias && ctx->needs_input_grad(2)};
    if (ctx->saved_data["residual"].toBool()) out[3] = grads[0];
    if (!grads[0].defined() || !(need[0] || need[1] || need[2])) return out;
    {
      const at::NoGradGuard off;
      const auto saved = ctx->get_saved_variables();
      const at::Tensor &x = saved[0], &w = saved[1], gy = grads[0].resolve_neg().contiguous();
      c10::cuda::CUDAGuard guard(x.device());
      Layer l;
      describe_layer(&l, x, w, static_cast<int>(ctx->saved_data["act"].toInt()));
      if (need[0]) out[0] = at::empty(x.sizes(), x.options());
      if (need[1]) out[1] = at::empty(l.a.w_transposed ? std::vector<int64_t>{l.a.n, l.a.k} : std::vector<int64_t>{l.a.k, l.a.n}, x.options());
      if (need[2]) out[2] = at::empty({l.a.n}, x.options());
      l.a.gy = ptr(gy), l.a.z = ptr(saved[2]), l.a.gx = ptr(out[0]), l.a.gw = ptr(out[1]), l.a.gb = ptr(out[2]);
      const at::Tensor space = workspace(gelib_linear_workspace(&l.a, 1), x);
      void* s = stream_of(x.device());
      call([&] { return gelib_linear_back(&l.a, ptr(space), s); });
      if (need[1] && l.a.w_transposed) out[1] = out[1].t();
    }
    const at::Tensor residual = out[3];
    out[3] = at::Tensor();
    out = differentiable_once(std::move(out), "linear");
    out[3] = residual;
    return out;
  }
};

std::optional<at::Tensor> linear(const at::Tensor& x, const at::Tensor& w, const OptTensor& bias, const OptTensor& residual, int act) {
  if (!is_plain(x) || x.dim() < 1 || !w.defined() || w.dim() != 2 || x.size(-1) != w.size(0) || !goes_with(x, w, w.sizes())) return std::nullopt;
  if (w.size(0) > INT_MAX || w.size(1) > INT_MAX) return std::nullopt;
  c10::SmallVector<int64_t, 6> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = w.size(1);
  if (!goes_with(x, bias, {w.size(1)}) || !goes_with(x, residual, shape)) return std::nullopt;
  const at::Tensor b = or_none(bias), r = or_none(residual);
  const auto wants = [](const at::Tensor& t) { return t.defined() && t.requires_grad(); };
  if (at::GradMode::is_enabled() && (wants(x) || wants(w) || wants(b) || wants(r))) return LinearFunction::apply(x, w, bias, residual, static_cast<int64_t>(act));
  Layer l;
  return linear_call(&l, x, w, b, r, act, false);
}

struct NormSizes {
  int64_t b, s;
  int n, type;
};
NormSizes norm_sizes(const at::Tensor& x) {
  NormSizes z = {x.size(0), 1, static_cast<int>(x.size(-1)), *type_code(x.scalar_type())};
  for (int64_t d = 1; d + 1 < x.dim(); d++) z.s *= x.size(d);
  return z;
}

// stats: (2, b, groups) for the means and the inverse deviations, or undefined.
at::Tensor norm_call(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& bias, int groups, double eps, int act, const at::Tensor& stats) {
  c10::cuda::CUDAGuard guard(x.device());
  const NormSizes z = norm_sizes(x);
  const at::Tensor y = at::empty(x.sizes(), x.options()), space = workspace(gelib_group_norm_workspace(z.b, z.s, z.n, groups, z.type, 0), x);
  float* mean = stats.defined() ? stats.data_ptr<float>() : nullptr;
  void* s = stream_of(x.device());
  call([&] {
    return gelib_group_norm(ptr(y), mean, mean ? mean + z.b * groups : nullptr, ptr(x), ptr(weight), ptr(bias), z.b, z.s, z.n, groups, eps, act, z.type, ptr(space), s);
  });
  return y;
}

struct GroupNormFunction : torch::autograd::Function<GroupNormFunction> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const OptTensor& weight, const OptTensor& bias, int64_t groups, double eps, int64_t act) {
    const at::Tensor stats = at::empty({2, x.size(0), groups}, x.options().dtype(at::kFloat));
    at::Tensor y = norm_call(x, or_none(weight), or_none(bias), static_cast<int>(groups), eps, static_cast<int>(act), stats);
    ctx->save_for_backward({x, or_none(weight), or_none(bias), stats});
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["act"] = act;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(6);
    if (!grads[0].defined()) return out;
    {
      const at::NoGradGuard off;
      const auto saved = ctx->get_saved_variables();
      const at::Tensor &x = saved[0], &stats = saved[3], gy = grads[0].resolve_neg().contiguous();
      c10::cuda::CUDAGuard guard(x.device());
      const NormSizes z = norm_sizes(x);
      const int groups = static_cast<int>(ctx->saved_data["groups"].toInt()), act = static_cast<int>(ctx->saved_data["act"].toInt());
      for (int i = 0, edge = 0; i < 3; i++)   // edges are counted over the tensors that were given
        if (saved[i].defined() && ctx->needs_input_grad(edge++)) out[i] = at::empty(saved[i].sizes(), x.options());
      const at::Tensor space = workspace(gelib_group_norm_workspace(z.b, z.s, z.n, groups, z.type, 1), x);
      const float* mean = stats.data_ptr<float>();
      void* s = stream_of(x.device());
      call([&] {
        return gelib_group_norm_back(ptr(out[0]), ptr(out[1]), ptr(out[2]), ptr(gy), ptr(x), ptr(saved[1]), ptr(saved[2]), mean, mean + z.b * groups, z.b, z.s, z.n, groups,
                                     act, z.type, ptr(space), s);
      });
    }
    return differentiable_once(std::move(out), "group_norm");
  }
};

std::optional<at::Tensor> group_norm(const at::Tensor& x, int groups, const OptTensor& weight, const OptTensor& bias, double eps, int act) {
  if (!is_plain(x) || x.dim() < 2 || !x.is_contiguous() || x.size(-1) > INT_MAX || groups < 1 || x.size(-1) % groups) return std::nullopt;
  for (const OptTensor* t : {&weight, &bias})
    if (!goes_with(x, *t, {x.size(-1)}) || (*t && !(*t)->is_contiguous())) return std::nullopt;
  const at::Tensor w = or_none(weight), b = or_none(bias);
  const auto wants = [](const at::Tensor& t) { return t.defined() && t.requires_grad(); };
  if (at::GradMode::is_enabled() && (wants(x) || wants(w) || wants(b)))
    return GroupNormFunction::apply(x, weight, bias, static_cast<int64_t>(groups), eps, static_cast<int64_t>(act));
  return norm_call(x, w, b, groups, eps, act, at::Tensor());
}

// ---- embedding tables and losses ---------------------------------------------------------------------------------------------------

bool plain_numbers(const at::Tensor& t, c10::Device device) {
  return t.defined() && t.device() == device && t.layout() == at::kStrided && (t.scalar_type() == at::kLong || t.scalar_type() == at::kInt);
}

// state: for the gradient, or undefined.
at::Tensor embedding_call(const at::Tensor& ids, const at::Tensor& w, double scale, int64_t padding, at::Tensor* state) {
  c10::cuda::CUDAGuard guard(w.device());
  const int64_t n = ids.numel(), d = w.size(1);
  const int v = static_cast<int>(w.size(0));
  c10::SmallVector<int64_t, 6> shape(ids.sizes().begin(), ids.sizes().end());
  shape.push_back(d);
  const at::Tensor y = at::empty(shape, w.options());
  if (state) *state = workspace(gelib_embedding_state_bytes(n, v), w);
  void *s = stream_of(w.device()), *kept = state ? ptr(*state) : nullptr;
  const int type = *type_code(w.scalar_type()), bytes = static_cast<int>(ids.element_size());
  call([&] { return gelib_embedding(ptr(y), ptr(ids), ptr(w), n, v, static_cast<int>(d), std::max(w.stride(0), d), scale, padding, bytes, type, kept, s); });
  return y;
}

struct EmbeddingFunction : torch::autograd::Function<EmbeddingFunction> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& ids, const at::Tensor& w, double scale, int64_t padding) {
    at::Tensor state, y = embedding_call(ids, w, scale, padding, &state);
    ctx->save_for_backward({state});
    ctx->saved_data["n"] = ids.numel();
    ctx->saved_data["v"] = w.size(0);
    ctx->saved_data["d"] = w.size(1);
    ctx->saved_data["scale"] = scale;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(4);
    if (!grads[0].defined()) return out;
    {
      const at::NoGradGuard off;
      const at::Tensor state = ctx->get_saved_variables()[0], gy = grads[0].resolve_neg().contiguous();
      c10::cuda::CUDAGuard guard(gy.device());
      const int64_t n = ctx->saved_data["n"].toInt();
      const int v = static_cast<int>(ctx->saved_data["v"].toInt()), d = static_cast<int>(ctx->saved_data["d"].toInt()), type = *type_code(gy.scalar_type());
      const double scale = ctx->saved_data["scale"].toDouble();
      out[1] = at::empty({v, d}, gy.options());
      const at::Tensor space = workspace(gelib_embedding_workspace(n, v, d, type), gy);
      void* s = stream_of(gy.device());
      call([&] { return gelib_embedding_back(ptr(out[1]), ptr(gy), ptr(state), n, v, d, scale, type, ptr(space), s); });
    }
    return differentiable_once(std::move(out), "embedding");
  }
};

std::optional<at::Tensor> embedding(const at::Tensor& ids, const at::Tensor& w, double scale, std::optional<int64_t> padding_idx) {
  if (!is_plain(w) || w.dim() != 2 || !plain_numbers(ids, w.device()) || !ids.is_contiguous() || ids.numel() == 0 || w.numel() == 0) return std::nullopt;
  const int64_t v = w.size(0), d = w.size(1);
  if (v > INT_MAX || d > INT_MAX || (w.stride(1) != 1 && d > 1) || (w.stride(0) < d && v > 1)) return std::nullopt;
  if (padding_idx && (*padding_idx < -v || *padding_idx >= v)) return std::nullopt;
  const int64_t padding = padding_idx ? (*padding_idx < 0 ? *padding_idx + v : *padding_idx) : -1;
  if (at::GradMode::is_enabled() && w.requires_grad()) return EmbeddingFunction::apply(ids, w, scale, padding);
  return embedding_call(ids, w, scale, padding, nullptr);
}

struct LossCall {
  gelib_linear_loss_args a = {};
  at::Tensor x, w;
};
// x and w as they lie, or copies; the rest is dense.
void describe_loss(LossCall* l, const at::Tensor& x, const at::Tensor& w, const at::Tensor& bias, const at::Tensor& target, const at::Tensor& teacher) {
  l->a.k = static_cast<int>(w.size(0));
  l->a.n = static_cast<int>(w.size(1));
  l->a.m = 1;
  for (int64_t d = 0; d + 1 < x.dim(); d++) l->a.m *= x.size(d);
  l->x = as_rows(x, l->a.k, &l->a.ldx);
  l->a.w_transposed = w.stride(0) == 1 && w.stride(1) != 1 && w.stride(1) >= l->a.k;
  if (l->a.w_transposed) l->w = w, l->a.ldw = w.stride(1);
  else l->w = as_rows(w, l->a.n, &l->a.ldw);
  l->a.x = ptr(l->x), l->a.w = ptr(l->w), l->a.bias = ptr(bias), l->a.target = ptr(target), l->a.teacher = ptr(teacher);
  l->a.top = teacher.defined() ? static_cast<int>(teacher.size(-1)) : 1;
  l->a.type = *type_code(x.scalar_type()), l->a.teacher_type = teacher.defined() ? *type_code(teacher.scalar_type()) : 0;
  l->a.index_bytes = static_cast<int>(target.element_size());
}

// state: what the backward call needs of it.
at::Tensor loss_call(LossCall* l, const at::Tensor& x, const at::Tensor& w, const at::Tensor& bias, const at::Tensor& target, const at::Tensor& teacher, at::Tensor* state) {
  c10::cuda::CUDAGuard guard(x.device());
  describe_loss(l, x, w, bias, target, teacher);
  const at::Tensor loss = at::empty(l->a.reduction == GELIB_LOSS_NONE ? x.sizes().slice(0, x.dim() - 1) : at::IntArrayRef{}, x.options().dtype(at::kFloat));
  *state = at::empty({gelib_linear_loss_state_bytes(&l->a)}, x.options().dtype(at::kByte));
  l->a.loss = ptr(loss), l->a.state = ptr(*state);
  const at::Tensor space = workspace(gelib_linear_loss_workspace(&l->a, 0), x);
  void* s = stream_of(x.device());
  call([&] { return gelib_linear_loss(&l->a, ptr(space), s); });
  return loss;
}

struct LinearLossFunction : torch::autograd::Function<LinearLossFunction> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w, const OptTensor& bias, const at::Tensor& target, const OptTensor& teacher,
                            int64_t reduction, int64_t ignore_index, double temperature) {
    LossCall l;
    l.a.reduction = static_cast<int>(reduction), l.a.ignore_index = ignore_index, l.a.temperature = temperature;
    at::Tensor state, loss = loss_call(&l, x, w, or_none(bias), target, or_none(teacher), &state);
    ctx->save_for_backward({x, w, or_none(bias), target, or_none(teacher), state});
    ctx->saved_data["reduction"] = reduction;
    ctx->saved_data["ignore_index"] = ignore_index;
    ctx->saved_data["temperature"] = temperature;
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(8);
    if (!grads[0].defined()) return out;
    const char* name;
    {
      const at::NoGradGuard off;
      const auto saved = ctx->get_saved_variables();
      name = saved[4].defined() ? "linear_distillation" : "linear_cross_entropy";
      const at::Tensor &x = saved[0], gy = grads[0].resolve_neg().contiguous();
      c10::cuda::CUDAGuard guard(x.device());
      LossCall l;
      l.a.reduction = static_cast<int>(ctx->saved_data["reduction"].toInt()), l.a.ignore_index = ctx->saved_data["ignore_index"].toInt();
      l.a.temperature = ctx->saved_data["temperature"].toDouble();
      describe_loss(&l, x, saved[1], saved[2], saved[3], saved[4]);
      // edges are counted over the tensors that were given
      if (ctx->needs_input_grad(0)) out[0] = at::empty(x.sizes(), x.options());
      if (ctx->needs_input_grad(1)) out[1] = at::empty(l.a.w_transposed ? std::vector<int64_t>{l.a.n, l.a.k} : std::vector<int64_t>{l.a.k, l.a.n}, x.options());
      if (saved[2].defined() && ctx->needs_input_grad(2)) out[2] = at::empty({l.a.n}, x.options());
      l.a.gy = ptr(gy), l.a.state = ptr(saved[5]), l.a.gx = ptr(out[0]), l.a.gw = ptr(out[1]), l.a.gb = ptr(out[2]);
      const at::Tensor space = workspace(gelib_linear_loss_workspace(&l.a, 1), x);
      void* s = stream_of(x.device());
      call([&] { return gelib_linear_loss_back(&l.a, ptr(space), s); });
      if (out[1].defined() && l.a.w_transposed) out[1] = out[1].t();
    }
    return differentiable_once(std::move(out), name);
  }
};

std::optional<at::Tensor> linear_loss(const at::Tensor& x, const at::Tensor& w, const OptTensor& bias, const at::Tensor& target, const OptTensor& teacher, int reduction,
                                      int64_t ignore_index, double temperature) {
  if (!is_plain(x) || x.dim() < 1 || x.numel() == 0 || !w.defined() || w.dim() != 2 || w.numel() == 0 || x.size(-1) != w.size(0) || !goes_with(x, w, w.sizes()))
    return std::nullopt;
  if (w.size(0) > INT_MAX || w.size(1) > INT_MAX || !goes_with(x, bias, {w.size(1)}) || (bias && !bias->is_contiguous())) return std::nullopt;
  if (!plain_numbers(target, x.device()) || !target.is_contiguous()) return std::nullopt;
  const auto lead = x.sizes().slice(0, x.dim() - 1);
  if (teacher) {
    const at::Tensor& t = *teacher;
    if (!is_plain(t) || t.device() != x.device() || !t.is_contiguous() || t.requires_grad() || t.dim() != x.dim() || t.sizes().slice(0, lead.size()) != lead) return std::nullopt;
    if (target.sizes() != t.sizes() || t.size(-1) < 1 || t.size(-1) > GELIB_LOSS_MAX_TOP) return std::nullopt;
  } else if (target.sizes() != lead) {
    return std::nullopt;
  }
  const at::Tensor b = or_none(bias);
  const auto wants = [](const at::Tensor& t) { return t.defined() && t.requires_grad(); };
  if (at::GradMode::is_enabled() && (wants(x) || wants(w) || wants(b)))
    return LinearLossFunction::apply(x, w, bias, target, teacher, static_cast<int64_t>(reduction), ignore_index, temperature);
  LossCall l;
  l.a.reduction = reduction, l.a.ignore_index = ignore_index, l.a.temperature = temperature;
  at::Tensor state;
  return loss_call(&l, x, w, b, target, or_none(teacher), &state);
}

}  // namespace

PYBIND11_MODULE(_native, m) {
  m.attr("torch_version") = GELIB_TORCH_VERSION;
  m.def("vec_forward", torch::wrap_pybind_function(&vec_forward));
  m.def("vec_backward", torch::wrap_pybind_function(&vec_backward));
  m.def("part_forward", torch::wrap_pybind_function(&part_forward));
  m.def("part_backward", torch::wrap_pybind_function(&part_backward));
  m.def("linear", torch::wrap_pybind_function(&linear));
  m.def("group_norm", torch::wrap_pybind_function(&group_norm));
  m.def("embedding", torch::wrap_pybind_function(&embedding));
  m.def("linear_loss", torch::wrap_pybind_function(&linear_loss));
  m.def("block8_values", torch::wrap_pybind_function(&block8_values));
  m.def("adamw_step", torch::wrap_pybind_function(&adamw_step));
  m.def("gather", torch::wrap_pybind_function(&gather));
}
