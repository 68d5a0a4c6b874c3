// The host side of the training-step operators where Python would take longer than the kernels.
//
// The optimiser step: reads every address, length and type of the parameters, gradients and states anew each step, straight
// from the tensors, hands them to the C entry points and marks what they write.  In Python the same walk costs 1.2 us per
// tensor (190 us for a network of 120 tensors whose kernels take 17 us); here 0.08 us.  The balance losses: argument checks,
// outputs, and the autograd nodes.
//
// A CPython extension compiled against torch's headers; it holds no CUDA code and calls libfsgs.so through the function
// pointers that bind() gives it.
#include <Python.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <unordered_map>
#include <utility>
#include <vector>

#include "../../include/fsgs.h"

namespace {

using AdamWFn = int (*)(int, const fsgs_adamw_tensor *, int, int, int, double, double, float, const float *, const float *,
    void *, size_t, fsgs_stream_t);
using NormFn = int (*)(int, const fsgs_norm_tensor *, float, void *, size_t, float *, fsgs_stream_t);

struct {
  AdamWFn adamw;
  NormFn norm;
  size_t (*norm_bytes)(void);
  size_t (*balance_bytes)(int64_t, int, int, int);
  int (*balance_count)(int64_t, int, int, const int64_t *, const uint8_t *, int, int64_t *, void *, size_t, fsgs_stream_t);
  int (*balance_pairs)(int64_t, int, int, const float *, const int64_t *, void *, size_t, float, const float *, float *, float *,
      int, fsgs_stream_t);
  int (*balance_table)(int64_t, int, int, const void *, int64_t, const uint8_t *, const int64_t *, void *, size_t, float,
      const float *, float *, void *, int64_t, fsgs_stream_t);
  const char *(*status_string)(int);
} lib;

// what a walk found, besides a status of the C entry points (0 or negative)
enum { kStale = 1, kStrided = 2 };

int type_of(at::ScalarType t) {
  return t == at::kFloat ? FSGS_F32 : t == at::kBFloat16 ? FSGS_BF16 : t == at::kHalf ? FSGS_F16 : -1;
}

struct StateTensor {
  PyObject *name;
  void *data;
  int64_t numel;
  at::ScalarType type;
  c10::TensorImpl *now;   // the tensor that the last walk found
  // still a dense tensor of that length and type there (the address tells the device): the kernels trust all of it
  bool is(c10::TensorImpl *x) const {
    return x->has_storage() && x->dtype() == c10::scalarTypeToTypeMeta(type) && x->numel() == numel && x->is_contiguous() &&
           (const char *) x->unsafe_storage().data() + x->storage_offset() * (int64_t) x->itemsize() == (const char *) data;
  }
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
  c10::Device device{at::kCPU};
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

// The exception that is being handled, as the Python error that torch's own calls raise for it (out of memory among them).
PyObject *failed() {
  torch::translate_exception_to_python(std::current_exception());
  return nullptr;
}

void need(bool ok, const char *what, const std::string &message) {
  if (!ok) throw std::runtime_error(std::string(what) + ": " + message);
}

// What a kernel writes counts as modified in place: a graph that has saved it then raises instead of using the new values.
void written(c10::TensorImpl *t) {
  if (!t->is_inference()) t->bump_version();
}

// The names of a parameter's state, and where in its table row the address goes.
struct Slot {
  const char *name;
  void *fsgs_adamw_tensor::*untyped;
  float *fsgs_adamw_tensor::*typed;
  PyObject *key;
};
Slot slots32[] = {{"step", nullptr, &fsgs_adamw_tensor::step, nullptr},
                  {"exp_avg", &fsgs_adamw_tensor::exp_avg, nullptr, nullptr},
                  {"exp_avg_sq", &fsgs_adamw_tensor::exp_avg_sq, nullptr, nullptr},
                  {"master", nullptr, &fsgs_adamw_tensor::master, nullptr}};
Slot slots8[] = {{"step", nullptr, &fsgs_adamw_tensor::step, nullptr},
                 {"exp_avg", &fsgs_adamw_tensor::exp_avg, nullptr, nullptr},
                 {"exp_avg_sq_root", &fsgs_adamw_tensor::exp_avg_sq, nullptr, nullptr},
                 {"exp_avg_scale", nullptr, &fsgs_adamw_tensor::exp_avg_scale, nullptr},
                 {"exp_avg_sq_root_scale", nullptr, &fsgs_adamw_tensor::exp_avg_sq_scale, nullptr},
                 {"master", nullptr, &fsgs_adamw_tensor::master, nullptr}};

// One parameter: checks it, its gradient and its state, and fills its table row (but the rates).
Entry entry_of(PyObject *param, Py_ssize_t group, PyObject *state, bool master, int bits, fsgs_adamw_tensor *row, c10::Device device) {
  constexpr const char *what = "AdamW";
  need(THPVariable_Check(param), what, "parameters are tensors");
  const at::Tensor &t = THPVariable_Unpack(param);
  need(t.is_cuda() && t.device() == device, what, "CUDA parameters on one device");
  need(t.layout() == at::kStrided && t.is_contiguous() && type_of(t.scalar_type()) >= 0, what,
       "contiguous float32, bfloat16 or float16 parameters");
  const at::Tensor &g = t.grad();
  need(g.defined() && g.layout() == at::kStrided && (g.scalar_type() == t.scalar_type() || g.scalar_type() == at::kFloat), what,
       "a dense gradient of its parameter's type or float32");
  need(g.numel() == t.numel() && g.device() == device, what, "a gradient has another size or device than its parameter");
  Entry e{param, state, group, t.data_ptr(), t.numel(), t.scalar_type(), g.scalar_type(), {}, row};
  row->param = e.data, row->numel = e.numel;
  Slot *slots = bits == 8 ? slots8 : slots32;
  const int n = (bits == 8 ? 6 : 4) - (master ? 0 : 1);
  e.held.reserve((size_t) n);
  for (int k = 0; k < n; ++k) {
    Slot &s = slots[k];
    if (!s.key) s.key = PyUnicode_InternFromString(s.name);
    PyObject *v = PyDict_GetItem(state, s.key);
    need(v && THPVariable_Check(v), what, std::string("a parameter's state has no ") + s.name);
    const at::Tensor &x = THPVariable_Unpack(v);
    const bool scale = bits == 8 && (k == 3 || k == 4), moment = k == 1 || k == 2;
    const int64_t size = k == 0 ? 1 : scale ? (e.numel + FSGS_ADAMW_BLOCK - 1) / FSGS_ADAMW_BLOCK : e.numel;
    const at::ScalarType kind = bits == 8 && moment ? at::kFloat8_e4m3fn : at::kFloat;
    need(x.device() == device && x.layout() == at::kStrided && x.scalar_type() == kind && x.numel() == size && x.is_contiguous(), what,
         std::string("the state ") + s.name + " must be a contiguous " + c10::toString(kind) + " tensor of " + std::to_string(size) +
             " elements on the parameter's device");
    if (s.untyped) row->*s.untyped = x.data_ptr();
    else row->*s.typed = (float *) x.data_ptr();
    e.held.push_back({s.key, x.data_ptr(), size, kind, x.unsafeGetTensorImpl()});
  }
  return e;
}

// All tensors of a launch are updated at once, so none may be part of another, and a state belongs to one parameter.  Of the
// states the step counts are looked at: they tell a state, or a count, that was given to two parameters (all state tensors
// of 120 parameters: 18 us on top of a plan's 285, these 4).
void need_apart(const std::vector<Entry> &entries) {
  std::vector<std::pair<const char *, const char *>> spans;
  std::vector<const void *> steps;
  spans.reserve(entries.size()), steps.reserve(entries.size());
  for (const Entry &e : entries) {
    if (e.numel > 0) spans.emplace_back((const char *) e.data, (const char *) e.data + e.numel * c10::elementSize(e.type));
    steps.push_back(e.held[0].data);
  }
  std::sort(spans.begin(), spans.end());
  for (size_t i = 1; i < spans.size(); ++i) need(spans[i].first >= spans[i - 1].second, "AdamW", "two parameters share memory");
  std::sort(steps.begin(), steps.end());
  need(std::adjacent_find(steps.begin(), steps.end()) == steps.end(), "AdamW", "two parameters share a state");
}

// plan(entries, launches, bits): entries [(param, group, state, master, address of its table row)], launches
// [(n, address of the table, param type, gradient type, bits, beta1, beta2, eps)]
PyObject *make_plan(PyObject *, PyObject *args) {
  PyObject *entries, *launches;
  int bits;
  if (!PyArg_ParseTuple(args, "O!O!i", &PyList_Type, &entries, &PyList_Type, &launches, &bits)) return nullptr;
  auto *plan = new Plan;
  PyObject *capsule = PyCapsule_New(plan, "fsgs.plan", free_plan);
  if (!capsule) {
    delete plan;
    return nullptr;
  }
  plan->keep = PyTuple_Pack(2, entries, launches);
  plan->params_key = PyUnicode_InternFromString("params");
  const size_t count = (size_t) PyList_GET_SIZE(entries);
  plan->entries.reserve(count), plan->norm.reserve(count), plan->place.reserve(count);
  for (Py_ssize_t i = 0; i < PyList_GET_SIZE(entries); ++i) {
    PyObject *param, *state;
    Py_ssize_t group;
    int master;
    unsigned long long row;
    if (!PyArg_ParseTuple(PyList_GET_ITEM(entries, i), "OnO!pK", &param, &group, &PyDict_Type, &state, &master, &row)) {
      Py_DECREF(capsule);
      return nullptr;
    }
    try {
      if (i == 0 && THPVariable_Check(param)) plan->device = THPVariable_Unpack(param).device();
      plan->entries.push_back(entry_of(param, group, state, master, bits, (fsgs_adamw_tensor *) row, plan->device));
    } catch (...) {
      Py_DECREF(capsule);
      return failed();
    }
    const Entry &e = plan->entries.back();
    plan->place.emplace(param, plan->entries.size() - 1);
    plan->norm.push_back({nullptr, e.numel, type_of(e.grad_type)});
  }
  try {
    need_apart(plan->entries);
  } catch (...) {
    Py_DECREF(capsule);
    return failed();
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
      PyObject *name, *v;
      Py_ssize_t at = 0;
      bool in_order = true;  // a state's tensors mostly stand as they were put there
      for (StateTensor &h : e.held) {
        in_order = in_order && PyDict_Next(e.state, &at, &name, &v) && name == h.name;
        if (!in_order) v = PyDict_GetItem(e.state, h.name);
        if (!v || !THPVariable_Check(v) || !h.is(h.now = THPVariable_Unpack(v).unsafeGetTensorImpl())) return kStale;
      }
      e.row->grad = grad.data_ptr();
      plan.norm[i].data = e.row->grad;
      ++i;
    }
  }
  if (i != plan.entries.size()) return kStale;
  PyObject *key, *value;
  Py_ssize_t pos = 0;
  for (size_t next = 0; PyDict_Next(state, &pos, &key, &value);) {  // the states are still the parameters' states
    if (next >= plan.entries.size() || plan.entries[next].param != key) {  // mostly they come in the parameters' order
      auto it = plan.place.find(key);
      if (it == plan.place.end()) continue;
      next = it->second;
    }
    if (plan.entries[next++].state != value) return kStale;
    ++found;
  }
  return found != plan.entries.size() ? kStale : strided ? kStrided : 0;
}

void written(const Plan &plan) {
  for (const Entry &e : plan.entries) {
    written(THPVariable_Unpack(e.param).unsafeGetTensorImpl());
    for (const StateTensor &h : e.held) written(h.now);
  }
}

// The optimiser's own tensors, [(tensor, stream that it was made on)]: the allocator keeps them until this stream is done
// with them, should the optimiser be let go of meanwhile.
void keep_for(const c10::cuda::CUDAStream &stream, PyObject *own) {
  for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(own); ++i) {
    PyObject *pair = PyTuple_GET_ITEM(own, i);
    if ((cudaStream_t) PyLong_AsVoidPtr(PyTuple_GET_ITEM(pair, 1)) != stream.stream())
      THPVariable_Unpack(PyTuple_GET_ITEM(pair, 0)).record_stream(stream.unwrap());
  }
}

// step(plan, groups, state, max_norm, (norm workspace, its bytes, norm out, workspace, its bytes), own, grad_scale, gate): on
// the parameters' device and its current stream; addresses as integers, 0 for none; max_norm None: no norm
PyObject *step(PyObject *, PyObject *const *args, Py_ssize_t n) {
  if (n != 8 || !PyList_Check(args[1]) || !PyDict_Check(args[2]) || !PyTuple_Check(args[4]) || PyTuple_GET_SIZE(args[4]) != 5 ||
      !PyTuple_Check(args[5]))
    return refuse("fsgs_host.step: wrong arguments");
  Plan *plan = (Plan *) PyCapsule_GetPointer(args[0], "fsgs.plan");
  if (!plan) return nullptr;
  auto word = [&](int k) { return (uintptr_t) PyLong_AsUnsignedLongLong(PyTuple_GET_ITEM(args[4], k)); };
  const bool clip = args[3] != Py_None;
  const float max_norm = clip ? (float) PyFloat_AsDouble(args[3]) : 0.0f;
  void *norm_ws = (void *) word(0), *ws = (void *) word(3);
  const size_t norm_bytes = word(1), bytes = word(4);
  float *norm_out = clip ? (float *) word(2) : nullptr;
  const float *grad_scale = (const float *) (uintptr_t) PyLong_AsUnsignedLongLong(args[6]);
  const float *gate = (const float *) (uintptr_t) PyLong_AsUnsignedLongLong(args[7]);
  if (PyErr_Occurred()) return nullptr;
  try {
    int rc = walk(*plan, args[1], args[2]);
    if (rc != 0) return PyLong_FromLong(rc);
    written(*plan);
    const c10::cuda::CUDAGuard guard(plan->device);
    const auto current = c10::cuda::getCurrentCUDAStream(plan->device.index());
    const auto stream = (fsgs_stream_t) current.stream();
    keep_for(current, args[5]);
    if (norm_out) {
      rc = lib.norm((int) plan->norm.size(), plan->norm.data(), max_norm, norm_ws, norm_bytes, norm_out, stream);
      grad_scale = norm_out + 1;
    }
    for (const Launch &l : plan->launches) {
      if (rc != 0) break;
      rc = lib.adamw(l.n, l.table, l.param_type, l.grad_type, l.bits, l.b1, l.b2, l.eps, grad_scale, gate, ws, bytes, stream);
    }
    return PyLong_FromLong(rc);
  } catch (...) {
    return failed();
  }
}

fsgs_stream_t stream_of(const at::Tensor &t) { return (fsgs_stream_t) c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

PyObject *tuple_of(std::initializer_list<at::Tensor> list) {
  PyObject *out = PyTuple_New((Py_ssize_t) list.size());
  Py_ssize_t i = 0;
  for (const at::Tensor &t : list) PyTuple_SET_ITEM(out, i++, THPVariable_Wrap(t));
  return out;
}

// norm(tensors, max_norm) -> (norm, factor)
PyObject *norm_of(PyObject *, PyObject *const *args, Py_ssize_t n) {
  if (n != 2 || !PyList_Check(args[0])) return refuse("fsgs_host.norm: wrong arguments");
  const float max_norm = (float) PyFloat_AsDouble(args[1]);
  if (PyErr_Occurred()) return nullptr;
  try {
    const at::NoGradGuard none;
    const Py_ssize_t count = PyList_GET_SIZE(args[0]);
    need(count > 0, "grad_norm", "no tensors");
    std::vector<fsgs_norm_tensor> table((size_t) count);
    std::vector<at::Tensor> kept;
    c10::Device device(at::kCPU);
    for (Py_ssize_t i = 0; i < count; ++i) {
      PyObject *o = PyList_GET_ITEM(args[0], i);
      const bool tensor = THPVariable_Check(o);
      if (tensor && i == 0) device = THPVariable_Unpack(o).device();
      need(tensor && THPVariable_Unpack(o).is_cuda() && THPVariable_Unpack(o).device() == device &&
               THPVariable_Unpack(o).layout() == at::kStrided && type_of(THPVariable_Unpack(o).scalar_type()) >= 0,
           "grad_norm", "dense float32, bfloat16 or float16 CUDA tensors on one device");
    }
    const c10::cuda::CUDAGuard guard(device);
    for (Py_ssize_t i = 0; i < count; ++i) {
      const at::Tensor &t = THPVariable_Unpack(PyList_GET_ITEM(args[0], i));
      const at::Tensor *d = &t;
      if (!t.is_contiguous()) {
        kept.push_back(t.contiguous());
        d = &kept.back();
      }
      table[(size_t) i] = {d->data_ptr(), d->numel(), type_of(d->scalar_type())};
    }
    const auto options = at::TensorOptions().device(device);
    const int64_t bytes = (int64_t) lib.norm_bytes();
    at::Tensor out = at::empty({2}, options.dtype(at::kFloat)), ws = at::empty({bytes}, options.dtype(at::kByte));
    const int rc = lib.norm((int) count, table.data(), max_norm, ws.data_ptr(), (size_t) bytes, out.data_ptr<float>(), stream_of(out));
    need(rc == 0, "fsgs_grad_norm", std::string(lib.status_string(rc)) + " (status " + std::to_string(rc) + ")");
    return tuple_of({out.select(0, 0), out.select(0, 1)});
  } catch (...) {
    return failed();
  }
}

// ---- balance losses -----------------------------------------------------------------------------------------

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void check(int rc, const char *what) {
  if (rc != 0) throw std::runtime_error(std::string(what) + ": " + lib.status_string(rc) + " (status " + std::to_string(rc) + ")");
}

constexpr const char *kPairs = "balance_loss", *kTable = "table_balance_loss";

void check_rows(const char *what, const Tensor &rows, const Tensor &idx, int64_t M, const std::optional<Tensor> &mask) {
  need(lib.balance_count, what, "the library is not bound");
  need(rows.is_cuda() && rows.layout() == at::kStrided && rows.dim() == 2, what, "a two-dimensional CUDA tensor is expected");
  need(idx.dim() == 2 && idx.layout() == at::kStrided && idx.scalar_type() == at::kLong && idx.size(0) == rows.size(0) &&
           idx.size(1) > 0 && idx.size(1) <= INT32_MAX && idx.device() == rows.device(),
       what, "idx must be int64 [N,K] on the same device");
  need(M > 0 && M < INT32_MAX, what, "the number of superpoints must be positive");
  if (mask)
    need((mask->scalar_type() == at::kBool || mask->scalar_type() == at::kByte) && mask->layout() == at::kStrided &&
             mask->dim() == 1 && mask->size(0) == rows.size(0) && mask->device() == rows.device(),
         what, "mask must be bool [N] on the same device");
}

void check_pairs(const Tensor &weights, const Tensor &idx, int64_t M, const std::optional<Tensor> &mask) {
  check_rows(kPairs, weights, idx, M, mask);
  need(weights.scalar_type() == at::kFloat && weights.sizes() == idx.sizes(), kPairs, "weights must be float32 [N,K]");
}

int check_table(const Tensor &table, const Tensor &idx, const std::optional<Tensor> &mask) {
  check_rows(kTable, table, idx, table.dim() == 2 ? table.size(1) : 0, mask);
  const int type = type_of(table.scalar_type());
  need(type >= 0, kTable, "float32, bfloat16 or float16 table");
  return type;
}

const uint8_t *bytes_of(const std::optional<Tensor> &mask) { return mask ? (const uint8_t *) mask->data_ptr() : nullptr; }
std::optional<Tensor> dense(const std::optional<Tensor> &mask) { return mask ? std::optional<Tensor>(mask->contiguous()) : mask; }
struct Counted {
  Tensor counts, ws;  // counts [M + 4], and M more for a copy where one is asked for
  int64_t M;
};

Counted count(const char *what, const Tensor &idx, int64_t M, const std::optional<Tensor> &mask, int form, bool copy = false) {
  const size_t bytes = lib.balance_bytes(idx.size(0), (int) idx.size(1), (int) M, form);
  need(bytes > 0, what, "more than 2^36 pairs or table entries");
  Counted c{at::empty({M + 4 + (copy ? M : 0)}, idx.options()), at::empty({(int64_t) bytes}, idx.options().dtype(at::kByte)), M};
  const Tensor i = idx.contiguous();
  check(lib.balance_count(i.size(0), (int) i.size(1), (int) M, i.data_ptr<int64_t>(), bytes_of(mask), form,
                          c.counts.data_ptr<int64_t>(), c.ws.data_ptr(), bytes, stream_of(i)),
        "fsgs_balance_count");
  return c;
}

void pairs(int64_t N, int64_t K, const Counted &c, const float *weights, float scale, const float *upstream, float *loss, float *grad,
    bool accumulate) {
  check(lib.balance_pairs(N, (int) K, (int) c.M, weights, c.counts.data_ptr<int64_t>(), c.ws.data_ptr(),
                          (size_t) c.ws.numel(), scale, upstream, loss, grad, accumulate, stream_of(c.ws)),
        "fsgs_balance_pairs");
}

// counts: for the loss alone
void table_pass(const Tensor &t, int type, const std::optional<Tensor> &mask, const int64_t *counts, const Tensor &ws, float scale,
    const float *upstream, float *loss, void *grad) {
  const int64_t N = t.size(0), M = t.size(1);
  check(lib.balance_table(N, (int) M, type, t.data_ptr(), N > 1 ? t.stride(0) : M, bytes_of(mask), counts, ws.data_ptr(),
                          (size_t) ws.numel(), scale, upstream, loss, grad, M, stream_of(ws)),
        "fsgs_balance_table");
}

// the table itself where its rows are runs of memory that do not overlap, else a copy
Tensor rows_of(const Tensor &t) {
  return (t.stride(1) == 1 || t.size(1) == 1) && t.stride(0) >= t.size(1) ? t : t.contiguous();
}

// A backward pass is not differentiable itself: a graph through it raises when it is used.
Tensor once(const Tensor &grad, const Tensor &upstream) {
  if (!at::GradMode::is_enabled() || !upstream.requires_grad()) return grad;
  auto error = std::make_shared<torch::autograd::DelayedError>("the balance losses have no second derivatives", 1);
  return (*error)({grad.detach().set_requires_grad(true)})[0];
}

// The engine hands a gradient over on the stream on which the node that takes it was made, and a leaf keeps one node as long
// as any graph of it lives.  Under capture, with that node from a stream outside the capture, the hand-over would end the
// capture with an error; so it is refused before, and the capture stays good.
void hand_over(const char *what) {
  const auto stream = c10::cuda::getCurrentCUDAStream();
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return;
  const auto node = torch::autograd::get_current_node();
  const auto next = node && node->num_outputs() ? node->next_edge(0).function : nullptr;
  const auto theirs = next ? next->stream() : std::nullopt;
  if (!theirs || *theirs == stream.unwrap()) return;
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  const bool known = cudaStreamIsCapturing(c10::cuda::CUDAStream(*theirs).stream(), &status) == cudaSuccess;
  if (!known) (void) cudaGetLastError();
  need(known && status == cudaStreamCaptureStatusActive, what,
       "a backward pass is being captured, but a graph made earlier on another stream still holds the input: let go of its "
       "loss first, or capture the value_and_grad form");
}

struct PairsLoss : torch::autograd::Function<PairsLoss> {
  static variable_list forward(AutogradContext *ctx, const Tensor &weights, const Tensor &idx, int64_t M, const std::optional<Tensor> &mask) {
    const c10::cuda::CUDAGuard guard(weights.device());
    const Tensor w = weights.contiguous();
    const Counted c = count(kPairs, idx, M, dense(mask), FSGS_BALANCE_PAIRS, true);
    Tensor loss = at::empty({}, w.options().requires_grad(false));
    pairs(idx.size(0), idx.size(1), c, w.data_ptr<float>(), 1.0f, nullptr, loss.data_ptr<float>(), nullptr, false);
    // the backward pass reads the counts: the caller, who may change what it is given, gets a copy (a part of the same tensor,
    // so the saved one goes where autograd does not compare versions)
    Tensor counts = c.counts.narrow(0, M + 4, M);
    if (cudaMemcpyAsync(counts.data_ptr(), c.counts.data_ptr(), sizeof(int64_t) * (size_t) M, cudaMemcpyDeviceToDevice,
                        (cudaStream_t) stream_of(c.ws)) != cudaSuccess) {
      (void) cudaGetLastError();
      check(FSGS_ERR_LAUNCH, "copy of the counts");
    }
    ctx->save_for_backward({c.ws});
    ctx->saved_data["counts"] = c.counts;
    ctx->saved_data["N"] = idx.size(0), ctx->saved_data["K"] = idx.size(1), ctx->saved_data["M"] = M;
    ctx->mark_non_differentiable({counts});
    return {loss, counts};
  }
  static variable_list backward(AutogradContext *ctx, variable_list g) {
    if (!g[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    const auto saved = ctx->get_saved_variables();
    const Counted c{ctx->saved_data["counts"].toTensor(), saved[0], ctx->saved_data["M"].toInt()};
    const c10::cuda::CUDAGuard guard(c.ws.device());
    hand_over(kPairs);
    const int64_t N = ctx->saved_data["N"].toInt(), K = ctx->saved_data["K"].toInt();
    Tensor grad = at::empty({N, K}, g[0].options().requires_grad(false));
    pairs(N, K, c, nullptr, 1.0f, g[0].data_ptr<float>(), nullptr, grad.data_ptr<float>(), false);
    return {once(grad, g[0]), Tensor(), Tensor(), Tensor()};
  }
};

struct TableLoss : torch::autograd::Function<TableLoss> {
  static variable_list forward(AutogradContext *ctx, const Tensor &table, const Tensor &idx, const std::optional<Tensor> &mask) {
    const c10::cuda::CUDAGuard guard(table.device());
    const Tensor t = rows_of(table);
    const auto m = dense(mask);
    const Counted c = count(kTable, idx, t.size(1), m, FSGS_BALANCE_TABLE);
    Tensor loss = at::empty({}, t.options().dtype(at::kFloat).requires_grad(false)), counts = c.counts.narrow(0, 0, t.size(1));
    table_pass(t, type_of(t.scalar_type()), m, c.counts.data_ptr<int64_t>(), c.ws, 1.0f, nullptr, loss.data_ptr<float>(), nullptr);
    ctx->save_for_backward({t, m ? *m : Tensor(), c.ws});
    ctx->mark_non_differentiable({counts});
    return {loss, counts};
  }
  static variable_list backward(AutogradContext *ctx, variable_list g) {
    if (!g[0].defined()) return {Tensor(), Tensor(), Tensor()};
    const auto saved = ctx->get_saved_variables();
    const Tensor &t = saved[0];
    const c10::cuda::CUDAGuard guard(t.device());
    hand_over(kTable);
    Tensor grad = at::empty(t.sizes(), t.options().requires_grad(false));
    table_pass(t, type_of(t.scalar_type()), saved[1].defined() ? std::optional<Tensor>(saved[1]) : std::nullopt,
               nullptr, saved[2], 1.0f, g[0].data_ptr<float>(), nullptr, grad.data_ptr());
    return {once(grad, g[0]), Tensor(), Tensor()};
  }
};

bool tensor_of(PyObject *o, Tensor &t) {
  if (!THPVariable_Check(o)) return false;
  t = THPVariable_Unpack(o);
  return true;
}

std::optional<Tensor> mask_of(const char *what, PyObject *o) {
  if (o == Py_None) return std::nullopt;
  need(THPVariable_Check(o), what, "mask must be bool [N] on the same device");
  return THPVariable_Unpack(o);
}

// balance_pairs(weights, idx, M, mask, weight, grad, autograd) -> (loss, counts) or (loss, grad, counts)
PyObject *balance_pairs(PyObject *, PyObject *const *args, Py_ssize_t n) {
  if (n != 7) return refuse("fsgs_host.balance_pairs: wrong arguments");
  const int64_t M = PyLong_AsLongLong(args[2]);
  const float weight = (float) PyFloat_AsDouble(args[4]);
  if (PyErr_Occurred()) return nullptr;
  try {
    Tensor w, idx, grad;
    need(tensor_of(args[0], w) && tensor_of(args[1], idx), kPairs, "weights and idx must be tensors");
    const auto mask = mask_of(kPairs, args[3]);
    check_pairs(w, idx, M, mask);
    if (args[6] == Py_True) {
      const auto out = PairsLoss::apply(w, idx, M, mask);
      return tuple_of({out[0], out[1]});
    }
    const bool add = args[5] != Py_None;
    if (add)
      need(tensor_of(args[5], grad) && grad.sizes() == w.sizes() && grad.scalar_type() == at::kFloat && grad.is_contiguous() &&
               grad.device() == w.device(),
           "balance_value_and_grad", "grad must be contiguous float32 [N,K]");
    const c10::cuda::CUDAGuard guard(w.device());
    const at::NoGradGuard none;
    w = w.contiguous();
    const Counted c = count(kPairs, idx, M, dense(mask), FSGS_BALANCE_PAIRS);
    Tensor loss = at::empty({}, w.options().requires_grad(false));
    if (!add) grad = at::empty(w.sizes(), w.options().requires_grad(false));
    pairs(idx.size(0), idx.size(1), c, w.data_ptr<float>(), weight, nullptr, loss.data_ptr<float>(), grad.data_ptr<float>(), add);
    if (add) written(grad.unsafeGetTensorImpl());
    return tuple_of({loss, grad, c.counts.narrow(0, 0, M)});
  } catch (...) {
    return failed();
  }
}

// balance_table(table, idx, mask, weight, autograd) -> (loss, counts) or (loss, grad, counts)
PyObject *balance_table(PyObject *, PyObject *const *args, Py_ssize_t n) {
  if (n != 5) return refuse("fsgs_host.balance_table: wrong arguments");
  const float weight = (float) PyFloat_AsDouble(args[3]);
  if (PyErr_Occurred()) return nullptr;
  try {
    Tensor t, idx;
    need(tensor_of(args[0], t) && tensor_of(args[1], idx), kTable, "table and idx must be tensors");
    const auto mask = mask_of(kTable, args[2]);
    const int type = check_table(t, idx, mask);
    if (args[4] == Py_True) {
      const auto out = TableLoss::apply(t, idx, mask);
      return tuple_of({out[0], out[1]});
    }
    const c10::cuda::CUDAGuard guard(t.device());
    const at::NoGradGuard none;
    t = rows_of(t);
    const auto m = dense(mask);
    const Counted c = count(kTable, idx, t.size(1), m, FSGS_BALANCE_TABLE);
    Tensor loss = at::empty({}, t.options().dtype(at::kFloat).requires_grad(false));
    Tensor grad = at::empty(t.sizes(), t.options().requires_grad(false));
    table_pass(t, type, m, c.counts.data_ptr<int64_t>(), c.ws, weight, nullptr, loss.data_ptr<float>(), grad.data_ptr());
    return tuple_of({loss, grad, c.counts.narrow(0, 0, t.size(1))});
  } catch (...) {
    return failed();
  }
}

// bind(addresses): the entry points in the order of `lib`
PyObject *bind(PyObject *, PyObject *const *args, Py_ssize_t n) {
  constexpr Py_ssize_t count = sizeof(lib) / sizeof(void *);
  if (n != count) return refuse("fsgs_host.bind: wrong number of addresses");
  void *address[count];
  for (Py_ssize_t i = 0; i < count; ++i) address[i] = PyLong_AsVoidPtr(args[i]);
  if (PyErr_Occurred()) return nullptr;
  memcpy(&lib, address, sizeof(lib));
  Py_RETURN_NONE;
}

using Fast = PyObject *(*) (PyObject *, PyObject *const *, Py_ssize_t);
PyCFunction fast(Fast f) { return (PyCFunction) (void (*)(void)) f; }

PyMethodDef methods[] = {{"plan", make_plan, METH_VARARGS, nullptr},
                         {"step", fast(step), METH_FASTCALL, nullptr},
                         {"norm", fast(norm_of), METH_FASTCALL, nullptr},
                         {"balance_pairs", fast(balance_pairs), METH_FASTCALL, nullptr},
                         {"balance_table", fast(balance_table), METH_FASTCALL, nullptr},
                         {"bind", fast(bind), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fsgs_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fsgs_host(void) { return PyModule_Create(&module); }
