// Root-mean-square norm for autograd, without the interpreter in its forward or backward pass: a backward
// function in Python waits for the interpreter lock on the engine's thread, which for small layers is
// longer than everything else (5 x 37 rows of 1263, forward and backward with curvature, from Python 133 us).
//
// Arguments that the engine cannot take make rms_norm return None, and the caller finds out which and raises.
#include <Python.h>

#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <ATen/ops/zeros_like.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/kfac_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

decltype(&kfac_rms_norm) norm_entry = nullptr;
decltype(&kfac_rms_norm_backward_workspace_bytes) workspace_entry = nullptr;
decltype(&kfac_rms_norm_backward) backward_entry = nullptr;

int type_code(at::ScalarType t) {
  return t == at::kFloat ? 0 : t == at::kBFloat16 ? 1 : t == at::kHalf ? 2 : -1;
}
bool on_device(const Tensor& t) { return t.defined() && t.is_cuda() && t.layout() == at::kStrided; }

// rows of `dim` elements that lie side by side
Tensor rows_of(const Tensor& t, int64_t dim) {
  Tensor r = t.reshape({-1, dim});
  return dim > 1 && r.stride(1) != 1 ? r.contiguous() : r;
}
hipStream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

bool gain_ok(const Tensor& gain, const Tensor& x) {
  return !gain.defined() || (on_device(gain) && gain.device() == x.device() && gain.dim() == 1 &&
                             gain.size(0) == x.size(-1) && gain.is_contiguous() &&
                             (gain.scalar_type() == at::kFloat || gain.scalar_type() == x.scalar_type()));
}
// (the entry points take 32 bits of a row's length)
constexpr int64_t MAX_DIM = 1 << 24;
bool takes(const Tensor& x, const Tensor& residual, const Tensor& gain, const Tensor& curvature) {
  if (!on_device(x) || type_code(x.scalar_type()) < 0 || x.dim() < 1 || x.size(-1) < 1 || x.size(-1) > MAX_DIM)
    return false;
  if (residual.defined() && (!on_device(residual) || residual.device() != x.device() ||
                             residual.scalar_type() != x.scalar_type() || residual.sizes() != x.sizes()))
    return false;
  if (curvature.defined() && (!on_device(curvature) || curvature.device() != x.device() || curvature.dim() != 1 ||
                              curvature.size(0) != x.size(-1) || curvature.scalar_type() != at::kFloat ||
                              !curvature.is_contiguous()))
    return false;
  return gain_ok(gain, x);
}

void check(int status, const char* what) {
  TORCH_CHECK(status == KFAC_OK, what, " failed (code ", status, ")");
}
const void* address(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* writable(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }

struct Normed {
  Tensor y, h, scale;
};
Normed norm(const Tensor& x, const Tensor& residual, const Tensor& gain, double eps, bool eight) {
  const c10::DeviceGuard guard(x.device());      // (the handle of a null stream means that of the current device)
  const int64_t dim = x.size(-1);
  const Tensor rows = rows_of(x, dim), res = residual.defined() ? rows_of(residual, dim) : Tensor();
  Normed n;
  n.y = at::empty(x.sizes(), eight ? x.options().dtype(at::kFloat8_e4m3fn) : x.options());
  if (residual.defined()) n.h = at::empty(x.sizes(), x.options());
  if (eight) {
    auto sizes = x.sizes().vec();
    sizes.back() = 1;
    n.scale = at::empty(sizes, x.options().dtype(at::kFloat));
  }
  check(norm_entry(type_code(x.scalar_type()), gain.defined() && gain.scalar_type() == at::kFloat, rows.size(0), (int)dim,
                   address(rows), rows.stride(0), address(res), res.defined() ? res.stride(0) : 0, address(gain),
                   (float)eps, writable(n.y), writable(n.h), (float*)writable(n.scale), stream_of(x)),
        "kfac_rms_norm");
  return n;
}

struct RmsNorm : torch::autograd::Function<RmsNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& residual,
                               const std::optional<Tensor>& gain, double eps, const std::optional<Tensor>& curvature) {
    const Tensor res = residual.value_or(Tensor()), w = gain.value_or(Tensor());
    const Normed n = norm(x, res, w, eps, false);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({res.defined() ? n.h : x, w});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["curvature"] = curvature.value_or(Tensor());
    ctx->saved_data["residual"] = res.defined();
    if (res.defined()) return {n.y, n.h};
    return {n.y};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "rms_norm has no second derivative (create_graph)");
    const auto saved = ctx->get_saved_variables();
    const Tensor h = saved[0], gain = saved[1], curvature = ctx->saved_data["curvature"].toTensor();
    const bool residual = ctx->saved_data["residual"].toBool();
    const Tensor dy = grads[0], dh = residual ? grads[1] : Tensor();
    // (of the arguments of forward that are tensors, undefined ones are not counted)
    size_t at = 0;
    const bool need_x = ctx->needs_input_grad(at++);
    const bool need_res = residual && ctx->needs_input_grad(at++);
    const bool need_gain = gain.defined() && ctx->needs_input_grad(at++);
    const bool need_stream = need_x || need_res;
    Tensor dx, dgain;
    if (!dy.defined()) {
      dx = dh;
      if (curvature.defined()) curvature.zero_();
    } else {
      const int64_t dim = h.size(-1);
      const Tensor rows = rows_of(h, dim), d = rows_of(dy, dim);
      const int64_t n = rows.size(0);
      if (need_stream) dx = at::empty(h.sizes(), h.options());
      if (need_gain) dgain = at::empty_like(gain);
      if (n == 0) {
        if (dgain.defined()) dgain.zero_();
        if (curvature.defined()) curvature.zero_();
      } else if (need_stream || need_gain || curvature.defined()) {
        const Tensor dstream = need_stream && dh.defined() ? rows_of(dh, dim) : Tensor();
        const int type = type_code(h.scalar_type()), samples = h.dim() > 1 ? (int)h.size(0) : 1;
        Tensor scratch;
        size_t bytes = 0;
        if (dgain.defined() || curvature.defined()) {
          bytes = workspace_entry(type, n, (int)dim, samples, curvature.defined());
          scratch = at::empty({(int64_t)bytes}, h.options().dtype(at::kByte));
        }
        check(backward_entry(type, gain.defined() && gain.scalar_type() == at::kFloat, n, (int)dim, samples, address(d),
                             d.stride(0), address(dstream), dstream.defined() ? dstream.stride(0) : 0, address(rows),
                             rows.stride(0), address(gain), (float)ctx->saved_data["eps"].toDouble(), writable(dx),
                             writable(dgain), (float*)writable(curvature), writable(scratch), bytes, stream_of(h)),
              "kfac_rms_norm_backward");
        if (curvature.defined()) curvature.unsafeGetTensorImpl()->bump_version();
      }
    }
    return {need_x ? dx : Tensor(), need_res ? dx : Tensor(), dgain, Tensor(), Tensor()};
  }
};

// Other threads go on meanwhile: an allocation may free cached blocks, a launch wait for room in the stream's
// queue.
struct WithoutInterpreter {
  PyThreadState* const state = PyEval_SaveThread();
  ~WithoutInterpreter() { PyEval_RestoreThread(state); }
};

bool tensor_of(PyObject* o, Tensor& t) {
  if (o == Py_None) return true;
  if (!THPVariable_Check(o)) return false;
  t = THPVariable_Unpack(o);
  return true;
}
PyObject* tuple_of(const variable_list& tensors) {
  if (tensors.size() == 1) return THPVariable_Wrap(tensors[0]);
  PyObject* const r = PyTuple_New((Py_ssize_t)tensors.size());
  for (size_t i = 0; r && i < tensors.size(); ++i) {
    PyObject* const t = THPVariable_Wrap(tensors[i]);
    if (!t) {
      Py_DECREF(r);
      return nullptr;
    }
    PyTuple_SET_ITEM(r, (Py_ssize_t)i, t);
  }
  return r;
}

}  // namespace

// bind_norm(addresses of the three entry points)
PyObject* host_bind_norm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 3) {
    PyErr_SetString(PyExc_TypeError, "bind_norm(norm, workspace, backward)");
    return nullptr;
  }
  norm_entry = (decltype(norm_entry))PyLong_AsVoidPtr(args[0]);
  workspace_entry = (decltype(workspace_entry))PyLong_AsVoidPtr(args[1]);
  backward_entry = (decltype(backward_entry))PyLong_AsVoidPtr(args[2]);
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
}

// rms_norm(x, residual or None, gain or None, eps, curvature or None, eight bits) -> y or (y, h), with its
// backward pass; in 8 bits (y, scale) or (y, scale, h)
PyObject* host_rms_norm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 6) {
    PyErr_SetString(PyExc_TypeError, "rms_norm(x, residual, gain, eps, curvature, eight)");
    return nullptr;
  }
  const double eps = PyFloat_AsDouble(args[3]);
  const int eight = PyObject_IsTrue(args[5]);
  if (PyErr_Occurred()) return nullptr;
  try {
    Tensor x, residual, gain, curvature;
    if (!norm_entry || args[0] == Py_None || !tensor_of(args[0], x) || !tensor_of(args[1], residual) ||
        !tensor_of(args[2], gain) || !tensor_of(args[4], curvature) || !takes(x, residual, gain, curvature))
      Py_RETURN_NONE;
    for (const Tensor& t : {x, residual, gain})
      TORCH_CHECK(!t.defined() || !t._fw_grad(0).defined(), "rms_norm has no forward-mode derivative");
    const auto needs = [](const Tensor& t) { return t.defined() && t.requires_grad(); };
    variable_list out;
    {
      const WithoutInterpreter released;
      if (!eight && at::GradMode::is_enabled() && (needs(x) || needs(residual) || needs(gain))) {
        const auto maybe = [](const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; };
        out = RmsNorm::apply(x, maybe(residual), maybe(gain), eps, maybe(curvature));
      } else {
        const Normed n = norm(x, residual, gain, eps, eight);
        out = {n.y};
        if (n.scale.defined()) out.push_back(n.scale);
        if (n.h.defined()) out.push_back(n.h);
      }
    }
    return tuple_of(out);
  } catch (...) {
    torch::translate_exception_to_python(std::current_exception());      // (each as torch's own calls raise it)
    return nullptr;
  }
}
