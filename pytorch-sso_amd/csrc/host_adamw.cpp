// AdamW's update of a list of tensors: what the engine needs of them is looked up and checked here, without a loop in
// Python (for the 160 tensors of a ResNet-50 the checks and addresses of five lists).
//
// Arguments that the engine cannot take make adamw return False, and the caller finds out which and raises.
#include <Python.h>

#include <ATen/ops/empty.h>
#include <ATen/ops/empty_strided.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <vector>

#include "../../include/kfac_hip.h"

namespace {

using at::Tensor;

decltype(&kfac_adamw_batched) adamw_entry = nullptr;
decltype(&kfac_adamw_workspace_bytes) adamw_workspace_entry = nullptr;

constexpr int64_t STATE_BLOCK = 128;          // elements of an 8-bit state with one scale
constexpr double LEAST_EPS_8 = 1e-12;         // of updates with such states

int adamw_type(at::ScalarType t) {
  return t == at::kFloat ? 0 : t == at::kBFloat16 ? 1 : t == at::kHalf ? 2 : -1;
}

// `take(object, index)` for every object of a list or tuple; false where one of them is, or it is none
template <class F>
bool each_of(PyObject* o, F&& take) {
  if (!PyList_Check(o) && !PyTuple_Check(o)) return false;
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(o);
  for (Py_ssize_t i = 0; i < n; ++i)
    if (!take(PySequence_Fast_GET_ITEM(o, i), i)) return false;
  return true;
}
bool tensors_of(PyObject* o, std::vector<Tensor>& out) {
  return each_of(o, [&](PyObject* t, Py_ssize_t) {
    if (!THPVariable_Check(t)) return false;
    out.push_back(THPVariable_Unpack(t));
    return true;
  });
}
// States: tensors, or (numbers, scales)
bool states_of(PyObject* o, std::vector<Tensor>& numbers, std::vector<Tensor>& scales) {
  return each_of(o, [&](PyObject* t, Py_ssize_t) {
    if (THPVariable_Check(t)) {
      numbers.push_back(THPVariable_Unpack(t));
      return true;
    }
    std::vector<Tensor> both;
    if (!tensors_of(t, both) || both.size() != 2) return false;
    numbers.push_back(both[0]);
    scales.push_back(both[1]);
    return true;
  });
}

bool strided_on(const Tensor& t, at::Device device, at::ScalarType type) {
  return t.defined() && t.layout() == at::kStrided && t.device() == device && t.scalar_type() == type;
}
// The elements of `t` lie in memory as those of `like` do.
bool lies_as(const Tensor& t, const Tensor& like) {
  if (t.sizes() != like.sizes()) return false;
  for (int64_t d = 0; d < t.dim(); ++d)
    if (t.size(d) > 1 && t.stride(d) != like.stride(d)) return false;
  return true;
}

struct WithoutInterpreter {
  PyThreadState* const state = PyEval_SaveThread();
  ~WithoutInterpreter() { PyEval_RestoreThread(state); }
};

// A gradient is read where it is: its elements lie as its parameter's do, with their own sign.
bool read_in_place(const Tensor& grad, const Tensor& p) { return lies_as(grad, p) && !grad.is_neg(); }

// No element is written twice, or is one of a gradient that is read in place (another thread's, perhaps).
bool apart(const std::vector<Tensor>& written, const std::vector<Tensor>& params, const std::vector<Tensor>& grads) {
  typedef std::pair<const char*, const char*> Range;
  const auto range = [](const Tensor& t) {
    const char* const at = (const char*)t.const_data_ptr();
    return Range(at, at + t.numel() * (int64_t)t.element_size());
  };
  std::vector<Range> ranges;
  ranges.reserve(written.size());
  for (const Tensor& t : written)
    if (t.numel() > 0) ranges.push_back(range(t));
  std::sort(ranges.begin(), ranges.end());
  for (size_t i = 1; i < ranges.size(); ++i)
    if (ranges[i].first < ranges[i - 1].second) return false;
  for (size_t i = 0; i < grads.size(); ++i) {
    if (grads[i].numel() == 0 || !read_in_place(grads[i], params[i])) continue;
    const Range g = range(grads[i]);
    const auto behind = std::lower_bound(ranges.begin(), ranges.end(), Range(g.second, nullptr));
    if (behind != ranges.begin() && (behind - 1)->second > g.first) return false;
  }
  return true;
}

}  // namespace

// bind_adamw(addresses of the two entry points)
PyObject* host_bind_adamw(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 2) {
    PyErr_SetString(PyExc_TypeError, "bind_adamw(update, workspace)");
    return nullptr;
  }
  adamw_entry = (decltype(adamw_entry))PyLong_AsVoidPtr(args[0]);
  adamw_workspace_entry = (decltype(adamw_workspace_entry))PyLong_AsVoidPtr(args[1]);
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
}

// adamw(params, grads, m, v (tensors, or all of them (numbers, scales)), steps (a number, a list of numbers or a list of
// tensors), lr (a number or a tensor), beta1, beta2, eps, weight decay, seed) -> True, or False
PyObject* host_adamw(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 11) {
    PyErr_SetString(PyExc_TypeError, "adamw(params, grads, m, v, steps, lr, beta1, beta2, eps, weight_decay, seed)");
    return nullptr;
  }
  const bool lr_on_device = THPVariable_Check(args[5]);
  const double lr = lr_on_device ? 0. : PyFloat_AsDouble(args[5]), beta1 = PyFloat_AsDouble(args[6]),
               beta2 = PyFloat_AsDouble(args[7]), eps = PyFloat_AsDouble(args[8]), decay = PyFloat_AsDouble(args[9]);
  const unsigned long long seed = PyLong_AsUnsignedLongLongMask(args[10]);
  if (PyErr_Occurred()) return nullptr;
  try {
    std::vector<Tensor> params, grads, states[4], counters;
    if (!adamw_entry || !tensors_of(args[0], params) || !tensors_of(args[1], grads) || params.empty() ||
        !states_of(args[2], states[0], states[2]) || !states_of(args[3], states[1], states[3]))
      Py_RETURN_FALSE;
    const size_t n = params.size();
    const bool eight = !states[2].empty();
    if (grads.size() != n || states[0].size() != n || states[1].size() != n || states[2].size() != (eight ? n : 0) ||
        states[3].size() != (eight ? n : 0) || (eight && !(eps >= LEAST_EPS_8)))
      Py_RETURN_FALSE;
    const at::Device device = params[0].device();
    const at::ScalarType type = params[0].scalar_type();
    if (!params[0].is_cuda() || adamw_type(type) < 0) Py_RETURN_FALSE;
    // the numbers of the updates
    std::vector<int64_t> steps;
    if (PyLong_Check(args[4])) {
      steps.assign(n, PyLong_AsLongLong(args[4]));
    } else if (!tensors_of(args[4], counters)) {
      counters.clear();
      if (!each_of(args[4], [&](PyObject* t, Py_ssize_t) {
            steps.push_back(THPVariable_Check(t) ? 0 : PyLong_AsLongLong(t));
            return true;
          }))
        Py_RETURN_FALSE;
    }
    if (PyErr_Occurred()) {
      PyErr_Clear();
      Py_RETURN_FALSE;
    }
    if ((steps.empty() ? counters.size() : steps.size()) != n) Py_RETURN_FALSE;
    for (const int64_t t : steps)
      if (t < 1) Py_RETURN_FALSE;
    for (const Tensor& t : counters)
      if (!strided_on(t, device, at::kInt) || t.numel() != 1 || t.is_neg()) Py_RETURN_FALSE;
    Tensor rate;
    if (lr_on_device) {
      rate = THPVariable_Unpack(args[5]);
      if (counters.empty() || !strided_on(rate, device, at::kFloat) || rate.numel() != 1) Py_RETURN_FALSE;
    }
    const at::ScalarType state_types[4] = {eight ? at::kFloat8_e4m3fn : at::kFloat, eight ? at::kFloat8_e5m2 : at::kFloat,
                                           at::kFloat, at::kFloat};
    std::vector<Tensor> written(params);
    for (size_t i = 0; i < n; ++i) {
      const Tensor& p = params[i];
      if (!strided_on(p, device, type) || p.is_neg() || !p.unsafeGetTensorImpl()->is_non_overlapping_and_dense() ||
          !strided_on(grads[i], device, type) || grads[i].sizes() != p.sizes())
        Py_RETURN_FALSE;
      for (int k = 0; k < (eight ? 4 : 2); ++k) {
        const Tensor& t = states[k][i];
        if (!strided_on(t, device, state_types[k]) || t.is_neg()) Py_RETURN_FALSE;
        if (k < 2 ? !lies_as(t, p)
                  : t.dim() != 1 || !t.is_contiguous() || t.size(0) != (p.numel() + STATE_BLOCK - 1) / STATE_BLOCK)
          Py_RETURN_FALSE;
        written.push_back(t);
      }
    }
    written.insert(written.end(), counters.begin(), counters.end());
    if (!apart(written, params, grads)) Py_RETURN_FALSE;
    int status;
    {
      const WithoutInterpreter released;
      const c10::DeviceGuard guard(device);
      std::vector<int64_t> numel(n);
      std::vector<const void*> g(n);
      std::vector<void*> at[5];
      for (auto& a : at) a.resize(n);
      for (size_t i = 0; i < n; ++i) {
        Tensor& grad = grads[i];
        if (!read_in_place(grad, params[i])) {
          Tensor copy = at::empty_strided(params[i].sizes(), params[i].strides(), grad.options());
          copy.copy_(grad.detach());
          grad = copy;
        }
        numel[i] = params[i].numel();
        g[i] = grad.const_data_ptr();
        at[0][i] = params[i].mutable_data_ptr();
        for (int k = 0; k < (eight ? 4 : 2); ++k) at[1 + k][i] = states[k][i].mutable_data_ptr();
      }
      // (a view may have its sign still to be applied)
      if (rate.defined()) rate = rate.detach().resolve_neg();
      std::vector<int*> counter(counters.size());
      for (size_t i = 0; i < counters.size(); ++i) counter[i] = (int*)counters[i].mutable_data_ptr();
      Tensor scratch;
      const size_t bytes = adamw_workspace_entry((int)n, !counters.empty());
      if (bytes > 0) scratch = at::empty({(int64_t)bytes}, params[0].options().dtype(at::kByte).requires_grad(false));
      status = adamw_entry((int)n, numel.data(), adamw_type(type), eight ? 8 : 32, at[0].data(), g.data(), at[1].data(),
                           at[2].data(), eight ? (float* const*)at[3].data() : nullptr,
                           eight ? (float* const*)at[4].data() : nullptr, steps.empty() ? nullptr : steps.data(),
                           counters.empty() ? nullptr : counter.data(), lr,
                           rate.defined() ? (const float*)rate.const_data_ptr() : nullptr, beta1, beta2, eps, decay,
                           (unsigned)seed, scratch.defined() ? scratch.mutable_data_ptr() : nullptr, bytes,
                           c10::hip::getCurrentHIPStream(device.index()).stream());
    }
    TORCH_CHECK(status == KFAC_OK, "kfac_adamw_batched failed (code ", status, ")");
    // (a graph from before the update that goes through these is refused by its backward pass; inference tensors are in
    // no graph and have no version, and what has been updated is not to end in an error)
    for (const Tensor& t : written)
      if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
    Py_RETURN_TRUE;
  } catch (...) {
    torch::translate_exception_to_python(std::current_exception());      // (each as torch's own calls raise it)
    return nullptr;
  }
}
