// tilec._host: host code that reads torch tensors, where reading them from Python
// costs more than the kernels they are for.
//
//   adamw_step(params, grads, exp_avg, exp_avg_sq, copies, step, lr, beta1, beta2,
//              eps, weight_decay, grad_scale, stream_of) -> None
//   adamw_values_table(states)
//       -> None or (table, count, device, outputs)
//
// The first checks the lists, packs a tilec_adamw_tensor (include/tilec.h) for
// each parameter with a gradient and enqueues the step on stream_of(device), the
// handle of the current stream of the tensors' device.  The same checks attribute
// by attribute in Python take 1.1 us a tensor (80 us for 72 tensors, whose kernels
// take 12); these take 0.05.  What the step writes counts as modified in place
// for autograd.  The second packs the descriptions of tilec_adamw_values, whose
// float32 outputs it allocates, views of one storage.
//
//   layer_norm(x, weight, bias, eps, dtype, stream) -> (y, mean, rstd)
//   layer_norm_backward(dy, x, mean, rstd, weight, param_grads, stream)
//       -> (dx, dweight, dbias)
//
// check their arguments, allocate the outputs and enqueue the kernels on `stream`
// (the handle of the tensors' device's current stream): one row of 4096 then
// costs 6 us a call instead of 10.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include <algorithm>
#include <memory>
#include <string>
#include <vector>

#include "../../include/tilec.h"

namespace {

constexpr int64_t kBlock = 256;  // values per scale of an 8-bit state

struct Refused {
  PyObject* type;
  std::string what;
};

[[noreturn]] void bad_value(const std::string& what) { throw Refused{PyExc_ValueError, what}; }
[[noreturn]] void bad_type(const std::string& what) { throw Refused{PyExc_TypeError, what}; }

// A list or tuple, or whatever else is a sequence.
struct List {
  PyObject* seq;
  explicit List(PyObject* o) : seq(PySequence_Fast(o, "expected lists of tensors")) {
    if (seq == nullptr) throw python_error();
  }
  ~List() { Py_DECREF(seq); }
  List(const List&) = delete;
  Py_ssize_t size() const { return PySequence_Fast_GET_SIZE(seq); }
  PyObject* operator[](Py_ssize_t i) const { return PySequence_Fast_GET_ITEM(seq, i); }
};

const at::Tensor& tensor(const char* name, PyObject* o) {
  if (!THPVariable_Check(o)) bad_type(std::string(name) + " holds a " + Py_TYPE(o)->tp_name + ", expected tensors");
  return THPVariable_Unpack(o);
}

struct Reader {
  int64_t device = -1;

  // A dense tensor of n values on the parameters' GPU, of one of two types.
  const at::Tensor& read(const char* name, PyObject* o, int64_t n, at::ScalarType a, at::ScalarType b,
                         bool contiguous = true) {
    const at::Tensor& t = tensor(name, o);
    if (!t.is_cuda()) bad_type("needs tensors on a ROCm GPU (" + std::string(name) + " has one on " + t.device().str() + ")");
    if (t.layout() != at::kStrided) bad_type(std::string(name) + " has a tensor that is not dense");
    if (device < 0) device = t.get_device();
    if (t.get_device() != device) bad_type("needs all tensors on one ROCm GPU (" + std::string(name) + " has others)");
    if (t.scalar_type() != a && t.scalar_type() != b)
      bad_type(std::string(name) + " has a tensor of dtype " + toString(t.scalar_type()) + ", expected " + toString(a) +
               (a == b ? "" : std::string(" or ") + toString(b)));
    if (n >= 0 && t.numel() != n)
      bad_value(std::string(name) + " has a tensor of " + std::to_string(t.numel()) + " values, expected " + std::to_string(n));
    if (contiguous && !t.is_contiguous()) bad_value(std::string(name) + " has a tensor that is not contiguous");
    return t;
  }
};

int32_t code(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16 ? TILEC_BF16 : TILEC_F32; }

// Tensors that are written past torch: each is a new version of itself, so that a
// backward pass that saved the old one raises instead of reading the new.
// (Inference tensors have no versions.)
struct Written {
  std::vector<const at::Tensor*> all;
  void* add(const at::Tensor& t) {
    all.push_back(&t);
    return t.data_ptr();
  }
  void bump() const {
    for (const at::Tensor* t : all)
      if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
  }
};

// A state: its values or codes, and the scales of codes (bits 8).
void read_state(Reader& r, Written& w, const char* name, PyObject* o, int64_t n, at::ScalarType codes, int& bits,
                void*& values, float*& scales) {
  const bool pair = PyTuple_Check(o) || PyList_Check(o);
  if (bits == 0) bits = pair ? 8 : 32;
  if ((bits == 8) != pair) bad_value("states of 32 and of 8 bits are mixed");
  if (!pair) {
    values = w.add(r.read(name, o, n, at::kFloat, at::kFloat));
    return;
  }
  const List both(o);
  if (both.size() != 2) bad_value(std::string(name) + ": an 8-bit state is a pair (codes, scales)");
  values = w.add(r.read(name, both[0], n, codes, codes));
  scales = static_cast<float*>(w.add(r.read("scales", both[1], (n + kBlock - 1) / kBlock, at::kFloat, at::kFloat)));
}

PyObject* build_values(PyObject* const* args) {
  const List states(args[0]);
  const Py_ssize_t count = states.size();
  if (count == 0) Py_RETURN_NONE;
  Reader r;
  std::vector<tilec_adamw_tensor> table(count);
  int64_t total = 0;
  for (Py_ssize_t i = 0; i < count; ++i) {
    if (!PyTuple_Check(states[i]) && !PyList_Check(states[i])) bad_value("expected (codes, scales) pairs");
    const List both(states[i]);
    if (both.size() != 2) bad_value("expected (codes, scales) pairs");
    tilec_adamw_tensor& d = table[i];
    const at::Tensor& c = r.read("codes", both[0], -1, at::kChar, at::kByte);
    d.n = c.numel();
    const at::Tensor& s = r.read("scales", both[1], (d.n + kBlock - 1) / kBlock, at::kFloat, at::kFloat);
    const bool m = c.scalar_type() == at::kChar;
    (m ? d.exp_avg : d.exp_avg_sq) = c.data_ptr();
    (m ? d.exp_avg_scale : d.exp_avg_sq_scale) = static_cast<float*>(s.data_ptr());
    total += d.n;
  }
  const at::Tensor all =
      at::empty({total}, at::TensorOptions().dtype(at::kFloat).device(at::kCUDA, (c10::DeviceIndex)r.device));
  PyObject* outs = PyList_New(count);
  if (outs == nullptr) throw python_error();
  int64_t at = 0;
  for (Py_ssize_t i = 0; i < count; ++i) {
    const at::Tensor o = all.narrow(0, at, table[i].n);
    table[i].param = o.data_ptr();
    at += table[i].n;
    PyList_SET_ITEM(outs, i, THPVariable_Wrap(o));
  }
  return Py_BuildValue("(y#iLN)", reinterpret_cast<const char*>(table.data()),
                       (Py_ssize_t)(table.size() * sizeof(tilec_adamw_tensor)), (int)count, (long long)r.device, outs);
}

// A status of the library as the exception the ctypes binding raises for it.
void check(int rc) {
  if (rc == TILEC_OK) return;
  throw Refused{rc == TILEC_ERR_VALUE ? PyExc_ValueError : rc == TILEC_ERR_TYPE ? PyExc_TypeError : PyExc_RuntimeError,
                tilec_last_error()};
}

std::string shape(const at::Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + (t.dim() == 1 ? ",)" : ")");
}

// A tensor of one GPU, float32 or bfloat16.
struct OneGpu {
  int64_t device = -1;
  int32_t code(const char* name, const at::Tensor& t) {
    if (!t.is_cuda()) bad_type("needs tensors on a ROCm GPU (" + std::string(name) + " is on " + t.device().str() + ")");
    if (device < 0) device = t.get_device();
    if (t.get_device() != device) bad_type("needs all tensors on one GPU (" + std::string(name) + " is on another)");
    if (t.layout() != at::kStrided) bad_type(std::string(name) + " is not a dense tensor");
    if (t.scalar_type() != at::kFloat && t.scalar_type() != at::kBFloat16)
      bad_type("unsupported tensor " + std::string(name) + " of dtype " + toString(t.scalar_type()) +
               " (use float32 or bfloat16)");
    return ::code(t);
  }
};

// A matrix whose rows are contiguous (copied if they are not); one dimension is
// one row.
struct Rows {
  at::Tensor t;
  int64_t R, D, ld;
  Rows(const char* name, const at::Tensor& x) : t(x) {
    if (x.dim() != 1 && x.dim() != 2)
      bad_value("expected a 1-D or 2-D " + std::string(name) + ", got shape " + shape(x));
    R = x.dim() == 1 ? 1 : x.size(0);
    D = x.size(-1);
    if (D == 0) bad_value("rows without elements have no mean (shape " + shape(x) + ")");
    if ((D > 1 && x.stride(-1) != 1) || (R > 1 && x.stride(0) < D)) t = x.contiguous();
    ld = R > 1 ? t.stride(0) : D;
  }
};

at::Tensor vector(const char* name, const at::Tensor& t, int64_t n) {
  if (t.dim() != 1 || t.size(0) != n)
    bad_value(std::string(name) + " has shape " + shape(t) + ", expected (" + std::to_string(n) + ",)");
  return t.contiguous();
}

// weight or bias: absent, or [D] of one type for both.
struct Params {
  at::Tensor weight, bias;
  int32_t code = TILEC_F32;
  Params(OneGpu& gpu, PyObject* w, PyObject* b, int64_t D) {
    if (w != Py_None) {
      const at::Tensor& t = tensor("weight", w);
      code = gpu.code("weight", t);
      weight = vector("weight", t, D);
    }
    if (b != Py_None) {
      const at::Tensor& t = tensor("bias", b);
      const int32_t c = gpu.code("bias", t);
      if (w != Py_None && c != code) bad_type("weight and bias have different types");
      code = c;
      bias = vector("bias", t, D);
    }
  }
};

const void* data(const at::Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }

void* stream_of(PyObject* o) {
  void* s = PyLong_AsVoidPtr(o);
  if (s == nullptr && PyErr_Occurred()) throw python_error();
  return s;
}

double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}

PyObject* three(const at::Tensor& a, const at::Tensor& b, const at::Tensor& c) {
  PyObject* t = PyTuple_New(3);
  if (t == nullptr) throw python_error();
  const at::Tensor* all[3] = {&a, &b, &c};
  for (int i = 0; i < 3; ++i) {
    PyObject* o = all[i]->defined() ? THPVariable_Wrap(*all[i]) : nullptr;
    if (o == nullptr) Py_INCREF(o = Py_None);
    PyTuple_SET_ITEM(t, i, o);
  }
  return t;
}

// Memory that a step writes, given twice (a tied weight, one state for two
// parameters, overlapping views), would be a race between workgroups.  A value
// may go where it was read from: a copy that is its param, a gradient that is
// its copy, param or state.
//
// Every kind of tensor is a list of ranges, mostly in the order of their
// memory; the lists are merged and compared with the furthest end so far (72
// tensors with two states each: 0.4 us where the lists lie one behind another, 1
// where they interleave, 1.9 with one sort of all).
void refuse_overlaps(const std::vector<tilec_adamw_tensor>& table) {
  struct Range {
    uintptr_t lo, hi;
  };
  struct Kind {
    const char* name;
    Range *at, *end;
    bool sorted;
  };
  const size_t n = table.size();
  const std::unique_ptr<Range[]> room(new Range[7 * n]);
  Kind kinds[7] = {{"params"}, {"exp_avg"}, {"exp_avg_sq"}, {"copies"}, {"scales"}, {"scales"}, {"grads"}};
  const char* const grads = kinds[6].name;  // the kind that is only read
  for (int k = 0; k < 7; ++k) kinds[k].at = kinds[k].end = room.get() + k * n, kinds[k].sorted = true;
  auto put = [&](Kind& k, const void* p, int64_t bytes) {
    if (p == nullptr || bytes <= 0) return;
    const uintptr_t lo = reinterpret_cast<uintptr_t>(p);
    if (k.end != k.at && lo < k.end[-1].lo) k.sorted = false;
    *k.end++ = {lo, lo + (uintptr_t)bytes};
  };
  for (const auto& d : table) {
    const int64_t p = d.param_dtype == TILEC_BF16 ? 2 : 4, g = d.grad_dtype == TILEC_BF16 ? 2 : 4;
    const int64_t state = d.exp_avg_scale ? 1 : 4, scales = 4 * ((d.n + kBlock - 1) / kBlock);
    put(kinds[0], d.param, d.n * p);
    put(kinds[1], d.exp_avg, d.n * state);
    put(kinds[2], d.exp_avg_sq, d.n * state);
    if (d.copy != d.param || p != 2) put(kinds[3], d.copy, d.n * 2);
    put(kinds[4], d.exp_avg_scale, scales);
    put(kinds[5], d.exp_avg_sq_scale, scales);
    const bool in_place = (d.grad == d.param && g == p) || (d.grad == d.copy && g == 2) ||
                          ((d.grad == d.exp_avg || d.grad == d.exp_avg_sq) && g == state);
    if (!in_place) put(kinds[6], d.grad, d.n * g);
  }
  int left = 0;
  for (const Kind& k : kinds) {
    if (k.at == k.end) continue;
    if (!k.sorted) std::sort(k.at, k.end, [](const Range& a, const Range& b) { return a.lo < b.lo; });
    kinds[left++] = k;
  }
  uintptr_t written = 0, read = 0;  // furthest ends so far
  const char *writer = nullptr;     // whose
  while (left > 0) {
    Kind* next = kinds;
    for (Kind* k = kinds + 1; k < kinds + left; ++k)
      if (k->at->lo < next->at->lo) next = k;
    uintptr_t limit = UINTPTR_MAX;  // the others' first
    for (const Kind* k = kinds; k < kinds + left; ++k)
      if (k != next) limit = std::min(limit, k->at->lo);
    const bool writes = next->name != grads;
    do {
      const Range r = *next->at++;
      if (r.lo < written || (writes && r.lo < read)) {
        const std::string a = next->name, b = r.lo < written ? writer : grads;
        bad_value(a == b ? "two " + a + " share their memory" : a + " and " + b + " share their memory");
      }
      if (writes && r.hi > written) written = r.hi, writer = next->name;
      if (!writes) read = std::max(read, r.hi);
    } while (next->at != next->end && next->at->lo <= limit);
    if (next->at == next->end) *next = kinds[--left];
  }
}

PyObject* build_adamw(PyObject* const* args) {
  const List params(args[0]), grads(args[1]), m(args[2]), v(args[3]);
  const bool copied = args[4] != Py_None;
  const List copies(copied ? args[4] : params.seq);  // (an iterator gives its tensors once)
  const Py_ssize_t count = params.size();
  if (grads.size() != count || m.size() != count || v.size() != count || copies.size() != count)
    bad_value(std::to_string(count) + " params, " + std::to_string(grads.size()) + " grads, " +
              std::to_string(m.size()) + " and " + std::to_string(v.size()) + " states, " +
              std::to_string(copied ? copies.size() : count) + " copies");
  Reader r;
  Written w;
  int bits = 0;
  std::vector<tilec_adamw_tensor> table;
  std::vector<at::Tensor> kept;
  table.reserve(count);
  w.all.reserve(6 * count);
  for (Py_ssize_t i = 0; i < count; ++i) {
    if (grads[i] == Py_None) continue;
    tilec_adamw_tensor d{};
    const at::Tensor& p = r.read("params", params[i], -1, at::kFloat, at::kBFloat16);
    const int64_t n = p.numel();
    const at::Tensor* g = &r.read("grads", grads[i], n, at::kFloat, at::kBFloat16, false);
    if (!g->is_contiguous()) {
      kept.push_back(g->contiguous());
      g = &kept.back();
    }
    d.param = w.add(p);
    d.grad = g->const_data_ptr();
    d.param_dtype = code(p);
    d.grad_dtype = code(*g);
    d.n = n;
    read_state(r, w, "exp_avg", m[i], n, at::kChar, bits, d.exp_avg, d.exp_avg_scale);
    read_state(r, w, "exp_avg_sq", v[i], n, at::kByte, bits, d.exp_avg_sq, d.exp_avg_sq_scale);
    if (copied && copies[i] != Py_None) d.copy = w.add(r.read("copies", copies[i], n, at::kBFloat16, at::kBFloat16));
    table.push_back(d);
  }
  if (table.empty()) Py_RETURN_NONE;
  refuse_overlaps(table);
  const int64_t step = PyLong_AsLongLong(args[5]);
  if (step == -1 && PyErr_Occurred()) throw python_error();
  const double lr = number(args[6]), beta1 = number(args[7]), beta2 = number(args[8]), eps = number(args[9]),
               decay = number(args[10]);
  const float* grad_scale = nullptr;
  if (args[11] != Py_None) {
    const at::Tensor& t = r.read("grad_scale", args[11], -1, at::kFloat, at::kFloat, false);
    if (t.numel() != 1) bad_value("grad_scale has shape " + shape(t) + ", expected one value");
    grad_scale = static_cast<const float*>(t.const_data_ptr());
  }
  PyObject* stream = PyObject_CallFunction(args[12], "L", (long long)r.device);
  if (stream == nullptr) throw python_error();
  const THPObjectPtr held(stream);
  const c10::DeviceGuard guard(c10::Device(at::kCUDA, (c10::DeviceIndex)r.device));
  check(tilec_adamw(table.data(), (int32_t)table.size(), bits, step, lr, beta1, beta2, eps, decay, grad_scale,
                    stream_of(stream)));
  w.bump();
  Py_RETURN_NONE;
}

PyObject* build_norm(PyObject* const* args) {
  const at::Tensor& x = tensor("x", args[0]);
  OneGpu gpu;
  const int32_t x_code = gpu.code("x", x);
  const Rows r("x", x);
  const Params p(gpu, args[1], args[2], r.D);
  const double eps = number(args[3]);
  at::ScalarType type = x.scalar_type();
  if (args[4] != Py_None) {
    if (!THPDtype_Check(args[4])) bad_type("dtype is no torch.dtype");
    type = reinterpret_cast<THPDtype*>(args[4])->scalar_type;
    if (type != at::kFloat && type != at::kBFloat16)
      bad_type(std::string("unsupported dtype ") + toString(type) + " (use float32 or bfloat16)");
  }
  const c10::DeviceGuard guard(x.device());
  const at::Tensor y = at::empty(x.sizes(), x.options().dtype(type));
  const at::Tensor mean = at::empty({r.R}, x.options().dtype(at::kFloat)), rstd = at::empty_like(mean);
  check(tilec_layer_norm(r.t.const_data_ptr(), data(p.weight), data(p.bias), y.data_ptr(),
                         static_cast<float*>(mean.data_ptr()), static_cast<float*>(rstd.data_ptr()), r.R, r.D, r.ld,
                         r.D, x_code, code(y), p.code, (float)eps, stream_of(args[5])));
  return three(y, mean, rstd);
}

PyObject* build_norm_backward(PyObject* const* args) {
  const at::Tensor &dy = tensor("dy", args[0]), &x = tensor("x", args[1]);
  const at::Tensor &mean_in = tensor("mean", args[2]), &rstd_in = tensor("rstd", args[3]);
  OneGpu gpu;
  const int32_t y_code = gpu.code("dy", dy), x_code = gpu.code("x", x);
  if (dy.sizes() != x.sizes()) bad_value("dy has shape " + shape(dy) + ", x " + shape(x));
  const Rows d("dy", dy), r("x", x);
  for (const at::Tensor* t : {&mean_in, &rstd_in}) {
    gpu.code("mean and rstd", *t);
    if (t->scalar_type() != at::kFloat) bad_type("mean and rstd are float32");
  }
  const at::Tensor mean = vector("mean", mean_in, r.R), rstd = vector("rstd", rstd_in, r.R);
  const Params p(gpu, args[4], Py_None, r.D);
  const int sums = PyObject_IsTrue(args[5]);
  if (sums < 0) throw python_error();
  const c10::DeviceGuard guard(dy.device());
  const at::Tensor dx = at::empty(dy.sizes(), dy.options());
  at::Tensor dw, db, scratch;
  if (sums) {
    dw = at::empty({r.D}, dy.options().dtype(at::kFloat));
    db = at::empty_like(dw);
  }
  if (sums || r.R > 0) {
    const size_t need = tilec_layer_norm_backward_workspace_bytes(r.R, r.D, x_code);
    if (need > 0) scratch = at::empty({(int64_t)need}, dy.options().dtype(at::kByte));
    check(tilec_layer_norm_backward(
        d.t.const_data_ptr(), r.t.const_data_ptr(), static_cast<const float*>(mean.const_data_ptr()),
        static_cast<const float*>(rstd.const_data_ptr()), data(p.weight), dx.data_ptr(),
        sums ? static_cast<float*>(dw.data_ptr()) : nullptr, sums ? static_cast<float*>(db.data_ptr()) : nullptr, r.R,
        r.D, d.ld, r.ld, r.D, x_code, y_code, p.code, need > 0 ? scratch.data_ptr() : nullptr, need,
        stream_of(args[6])));
  }
  return three(dx, dw, db);
}

constexpr char kAdamw[] = "adamw_step", kValues[] = "adamw_values", kNorm[] = "layer_norm", kNormBackward[] = "layer_norm_backward";

template <PyObject* (*BUILD)(PyObject* const*), int ARGS, const char* NAME>
PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != ARGS) {
    PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", ARGS, count);
    return nullptr;
  }
  try {
    return BUILD(args);
  } catch (const Refused& e) {
    PyErr_SetString(e.type, (std::string(NAME) + ": " + e.what).c_str());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

template <PyObject* (*BUILD)(PyObject* const*), int ARGS, const char* NAME>
PyCFunction function() {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&call<BUILD, ARGS, NAME>));
}

PyMethodDef kMethods[] = {
    {"adamw_step", function<build_adamw, 13, kAdamw>(), METH_FASTCALL,
     "adamw_step(params, grads, exp_avg, exp_avg_sq, copies, step, lr, beta1, beta2, eps, weight_decay, grad_scale, "
     "stream_of)"},
    {"adamw_values_table", function<build_values, 1, kValues>(), METH_FASTCALL,
     "adamw_values_table(states) -> None or (table, count, device, outputs)"},
    {"layer_norm", function<build_norm, 6, kNorm>(), METH_FASTCALL,
     "layer_norm(x, weight, bias, eps, dtype, stream) -> (y, mean, rstd)"},
    {"layer_norm_backward", function<build_norm_backward, 7, kNormBackward>(), METH_FASTCALL,
     "layer_norm_backward(dy, x, mean, rstd, weight, param_grads, stream) -> (dx, dweight, dbias)"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&kModule); }
