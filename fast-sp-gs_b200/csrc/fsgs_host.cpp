// The host side of the optimiser step for many tensors: reads every address and length of the parameters, gradients and
// states anew each step, straight from the tensors, and hands them to the C entry points.  In Python the same walk costs
// 1.2 us per tensor (190 us for a network of 120 tensors whose kernels take 17 us); here 0.06 us.
//
// A CPython extension of two functions and a capsule, compiled against torch's headers; it holds no CUDA code and calls
// libfsgs.so through the function pointers that fsgs/optim.py gives it.
#include <Python.h>
#include <torch/csrc/autograd/python_variable.h>

#include <unordered_map>
#include <vector>

#include "../../include/fsgs.h"

namespace {

using AdamWFn = int (*)(int, const fsgs_adamw_tensor *, int, int, int, double, double, float, const float *, const float *,
    void *, size_t, fsgs_stream_t);
using NormFn = int (*)(int, const fsgs_norm_tensor *, float, void *, size_t, float *, fsgs_stream_t);

// what a walk found, besides a status of the C entry points (0 or negative)
enum { kStale = 1, kStrided = 2 };

int type_of(at::ScalarType t) {
  return t == at::kFloat ? FSGS_F32 : t == at::kBFloat16 ? FSGS_BF16 : t == at::kHalf ? FSGS_F16 : -1;
}

struct StateTensor {
  PyObject *name;
  void *data;
};

struct Entry {
  PyObject *param, *state;
  Py_ssize_t group;
  void *data;
  int64_t numel;
  at::ScalarType type, grad_type;
  std::vector<StateTensor> held;
  fsgs_adamw_tensor *row;
};

struct Launch {
  int n, param_type, grad_type, bits;
  fsgs_adamw_tensor *table;
  double b1, b2;
  float eps;
};

struct Plan {
  std::vector<Entry> entries;
  std::vector<Launch> launches;
  std::unordered_map<PyObject *, size_t> place;
  std::vector<fsgs_norm_tensor> norm;
  PyObject *keep = nullptr;   // the Python objects behind every pointer
  PyObject *params_key = nullptr;
};

void free_plan(PyObject *capsule) {
  Plan *p = (Plan *) PyCapsule_GetPointer(capsule, "fsgs.plan");
  if (!p) return;
  Py_XDECREF(p->keep);
  Py_XDECREF(p->params_key);
  delete p;
}

PyObject *refuse(const char *what) {
  PyErr_SetString(PyExc_RuntimeError, what);
  return nullptr;
}

// plan(entries, launches): entries [(param, group, state, names, address of its table row)], launches
// [(n, address of the table, param type, gradient type, bits, beta1, beta2, eps)]
PyObject *make_plan(PyObject *, PyObject *args) {
  PyObject *entries, *launches;
  if (!PyArg_ParseTuple(args, "O!O!", &PyList_Type, &entries, &PyList_Type, &launches)) return nullptr;
  auto *plan = new Plan;
  PyObject *capsule = PyCapsule_New(plan, "fsgs.plan", free_plan);
  if (!capsule) {
    delete plan;
    return nullptr;
  }
  plan->keep = PyTuple_Pack(2, entries, launches);
  plan->params_key = PyUnicode_InternFromString("params");
  for (Py_ssize_t i = 0; i < PyList_GET_SIZE(entries); ++i) {
    PyObject *param, *state, *names;
    Py_ssize_t group;
    unsigned long long row;
    if (!PyArg_ParseTuple(PyList_GET_ITEM(entries, i), "OnO!O!K", &param, &group, &PyDict_Type, &state, &PyTuple_Type, &names, &row)) {
      Py_DECREF(capsule);
      return nullptr;
    }
    if (!THPVariable_Check(param) || !THPVariable_Unpack(param).grad().defined()) {
      Py_DECREF(capsule);
      return refuse("AdamW: a parameter without a gradient");
    }
    const at::Tensor &t = THPVariable_Unpack(param);
    Entry e{param, state, group, t.data_ptr(), t.numel(), t.scalar_type(), t.grad().scalar_type(), {}, (fsgs_adamw_tensor *) row};
    for (Py_ssize_t k = 0; k < PyTuple_GET_SIZE(names); ++k) {
      PyObject *name = PyTuple_GET_ITEM(names, k), *v = PyDict_GetItem(state, name);
      if (!v || !THPVariable_Check(v)) {
        Py_DECREF(capsule);
        return refuse("AdamW: a parameter's state is incomplete");
      }
      e.held.push_back({name, THPVariable_Unpack(v).data_ptr()});
    }
    plan->place.emplace(param, plan->entries.size());
    plan->norm.push_back({nullptr, e.numel, type_of(e.grad_type)});
    plan->entries.push_back(std::move(e));
  }
  for (Py_ssize_t i = 0; i < PyList_GET_SIZE(launches); ++i) {
    Launch l;
    unsigned long long table;
    if (!PyArg_ParseTuple(PyList_GET_ITEM(launches, i), "iKiiiddf", &l.n, &table, &l.param_type, &l.grad_type, &l.bits, &l.b1, &l.b2, &l.eps)) {
      Py_DECREF(capsule);
      return nullptr;
    }
    l.table = (fsgs_adamw_tensor *) table;
    plan->launches.push_back(l);
  }
  return capsule;
}

// 0 where the plan still describes the parameters that have gradients, their states and their places; the gradients'
// addresses are then in the tables
int walk(Plan &plan, PyObject *groups, PyObject *state) {
  size_t i = 0, found = 0;
  bool strided = false;
  for (Py_ssize_t g = 0; g < PyList_GET_SIZE(groups); ++g) {
    PyObject *group = PyList_GET_ITEM(groups, g);
    PyObject *params = PyDict_Check(group) ? PyDict_GetItem(group, plan.params_key) : nullptr;
    if (!params || !PyList_Check(params)) return kStale;
    for (Py_ssize_t k = 0; k < PyList_GET_SIZE(params); ++k) {
      PyObject *p = PyList_GET_ITEM(params, k);
      if (!THPVariable_Check(p)) return kStale;
      const at::Tensor &t = THPVariable_Unpack(p);
      const at::Tensor &grad = t.grad();
      if (!grad.defined()) continue;
      if (i >= plan.entries.size()) return kStale;
      Entry &e = plan.entries[i];
      if (e.param != p || e.group != g || t.numel() != e.numel || t.scalar_type() != e.type || !t.is_contiguous() ||
          t.data_ptr() != e.data)
        return kStale;
      if (grad.scalar_type() != e.grad_type || grad.layout() != at::kStrided || grad.device() != t.device() || grad.numel() != e.numel)
        return kStale;
      strided = strided || !grad.is_contiguous();
      for (const StateTensor &h : e.held) {
        PyObject *v = PyDict_GetItem(e.state, h.name);
        if (!v || !THPVariable_Check(v) || THPVariable_Unpack(v).data_ptr() != h.data) return kStale;
      }
      e.row->grad = grad.data_ptr();
      plan.norm[i].data = e.row->grad;
      ++i;
    }
  }
  if (i != plan.entries.size()) return kStale;
  PyObject *key, *value;
  Py_ssize_t pos = 0;
  while (PyDict_Next(state, &pos, &key, &value)) {  // the states are still the parameters' states
    auto it = plan.place.find(key);
    if (it == plan.place.end()) continue;
    if (plan.entries[it->second].state != value) return kStale;
    ++found;
  }
  return found != plan.entries.size() ? kStale : strided ? kStrided : 0;
}

// step(plan, groups, state, adamw, norm, max_norm, norm workspace, its bytes, norm out, grad_scale, gate, workspace, its
// bytes, stream): addresses as integers, 0 for none; norm out 0: no norm
PyObject *step(PyObject *, PyObject *const *args, Py_ssize_t n) {
  if (n != 14 || !PyList_Check(args[1]) || !PyDict_Check(args[2])) return refuse("fsgs_host.step: wrong arguments");
  Plan *plan = (Plan *) PyCapsule_GetPointer(args[0], "fsgs.plan");
  if (!plan) return nullptr;
  auto at = [&](int k) { return (uintptr_t) PyLong_AsUnsignedLongLong(args[k]); };
  const auto adamw = (AdamWFn) at(3);
  const auto norm = (NormFn) at(4);
  const float max_norm = (float) PyFloat_AsDouble(args[5]);
  void *norm_ws = (void *) at(6), *ws = (void *) at(11);
  const size_t norm_bytes = at(7), bytes = at(12);
  float *norm_out = (float *) at(8);
  const float *grad_scale = (const float *) at(9), *gate = (const float *) at(10);
  const auto stream = (fsgs_stream_t) at(13);
  if (PyErr_Occurred()) return nullptr;
  int rc;
  try {
    rc = walk(*plan, args[1], args[2]);
  } catch (const std::exception &e) {
    return refuse(e.what());
  }
  if (rc != 0) return PyLong_FromLong(rc);
  if (norm_out) {
    rc = norm((int) plan->norm.size(), plan->norm.data(), max_norm, norm_ws, norm_bytes, norm_out, stream);
    if (rc != 0) return PyLong_FromLong(rc);
    grad_scale = norm_out + 1;
  }
  for (const Launch &l : plan->launches) {
    rc = adamw(l.n, l.table, l.param_type, l.grad_type, l.bits, l.b1, l.b2, l.eps, grad_scale, gate, ws, bytes, stream);
    if (rc != 0) break;
  }
  return PyLong_FromLong(rc);
}

// norm(tensors, norm, max_norm, workspace, its bytes, out, stream)
PyObject *norm_of(PyObject *, PyObject *const *args, Py_ssize_t n) {
  if (n != 7 || !PyList_Check(args[0])) return refuse("fsgs_host.norm: wrong arguments");
  auto at = [&](int k) { return (uintptr_t) PyLong_AsUnsignedLongLong(args[k]); };
  const auto norm = (NormFn) at(1);
  const float max_norm = (float) PyFloat_AsDouble(args[2]);
  void *ws = (void *) at(3);
  const size_t bytes = at(4);
  float *out = (float *) at(5);
  const auto stream = (fsgs_stream_t) at(6);
  if (PyErr_Occurred()) return nullptr;
  static const char *want = "grad_norm: dense float32, bfloat16 or float16 CUDA tensors on one device";
  try {
    const Py_ssize_t count = PyList_GET_SIZE(args[0]);
    std::vector<fsgs_norm_tensor> table((size_t) count);
    c10::Device device(at::kCPU);
    for (Py_ssize_t i = 0; i < count; ++i) {
      PyObject *o = PyList_GET_ITEM(args[0], i);
      if (!THPVariable_Check(o)) return refuse(want);
      const at::Tensor &t = THPVariable_Unpack(o);
      if (i == 0) device = t.device();
      const int type = type_of(t.scalar_type());
      if (!t.is_cuda() || t.device() != device || t.layout() != at::kStrided || type < 0) return refuse(want);
      if (!t.is_contiguous()) return PyLong_FromLong(kStrided);
      table[(size_t) i] = {t.data_ptr(), t.numel(), type};
    }
    return PyLong_FromLong(norm((int) count, table.data(), max_norm, ws, bytes, out, stream));
  } catch (const std::exception &e) {
    return refuse(e.what());
  }
}

PyMethodDef methods[] = {{"plan", make_plan, METH_VARARGS, nullptr},
                         {"step", (PyCFunction) (void (*)(void)) step, METH_FASTCALL, nullptr},
                         {"norm", (PyCFunction) (void (*)(void)) norm_of, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fsgs_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fsgs_host(void) { return PyModule_Create(&module); }
