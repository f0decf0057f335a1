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
//
//   rms_norm(x, weight, residual, eps, dtype) -> (y, h, rstd)
//   rms_norm_backward(dy, h, rstd, weight, dh, weight_grad) -> (dx, dweight)
//   quantize_fp8(x, block, dtype) -> (codes, scales)
//   dequantize_fp8(q, dtype) -> values
//   linear_fp8(x, weight, dtype, counters_of) -> out
//
// do the same and find the stream themselves; 8-bit operands are (codes, scales)
// pairs.
//
//   grad_norm(grads, max_norm, grad_scale, counters_of) -> (norm, scale)
//   clip_grads(grads, max_norm, grad_scale, counters_of) -> norm
//
// read lists as adamw_step does; counters_of(device index, stream, bytes) gives the
// zeroed counters that kernels leave zero.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#ifdef TILEC_TORCH_HIP  // this torch has GPU support
// (The headers of a torch for ROCm use this macro without defining it.)
#ifndef TORCH_CUDA_CPP_API
#define TORCH_CUDA_CPP_API
#endif
#include <ATen/cuda/EmptyTensor.h>
#include <c10/hip/HIPStream.h>
#endif
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include <algorithm>
#include <cmath>
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

// A tuple of tensors, None for those that are not defined.
PyObject* tuple(std::initializer_list<at::Tensor> all) {
  PyObject* t = PyTuple_New((Py_ssize_t)all.size());
  if (t == nullptr) throw python_error();
  Py_ssize_t i = 0;
  for (const at::Tensor& x : all) {
    PyObject* o = x.defined() ? THPVariable_Wrap(x) : nullptr;
    if (o == nullptr) Py_INCREF(o = Py_None);
    PyTuple_SET_ITEM(t, i++, o);
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
  return tuple({y, mean, rstd});
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
  return tuple({dx, dw, db});
}

// The type that an argument names; `other` where it is None.
at::ScalarType dtype(PyObject* o, at::ScalarType other) {
  if (o == Py_None) return other;
  if (!THPDtype_Check(o)) bad_type("dtype is no torch.dtype");
  return reinterpret_cast<THPDtype*>(o)->scalar_type;
}

bool is_wide(at::ScalarType t) { return t == at::kFloat || t == at::kBFloat16; }
bool is_fp8(at::ScalarType t) { return t == at::kFloat8_e4m3fn || t == at::kFloat8_e5m2; }

int32_t code_of(at::ScalarType t) {
  return t == at::kFloat ? TILEC_F32 : t == at::kBFloat16 ? TILEC_BF16 : t == at::kFloat8_e4m3fn ? TILEC_F8E4M3 : TILEC_F8E5M2;
}

constexpr int64_t kGroup = 128;                      // values of a row under one scale of an 8-bit operand
constexpr int64_t kMaxScaleRow = int64_t(1) << 21;  // the largest row stride of scales in a product
int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// The current stream of a GPU, and a new tensor on one, past the dispatcher: 0.5 us
// instead of 0.75.  (A torch without GPU support has no tensor that gets here.)
#ifdef TILEC_TORCH_HIP
void* stream_on(at::Device device) { return c10::hip::getCurrentHIPStream(device.index()).stream(); }
at::Tensor make(at::IntArrayRef sizes, at::ScalarType type, at::Device device) {
  return at::Tensor(at::detail::empty_cuda(sizes, type, device, std::nullopt));
}
#else
void* stream_on(at::Device) { bad_type("needs a torch with GPU support"); }
at::Tensor make(at::IntArrayRef, at::ScalarType, at::Device) { bad_type("needs a torch with GPU support"); }
#endif

// The zeroed counters, which kernels leave zero, that `counters_of` gives.
at::Tensor zeroed(PyObject* counters_of, at::Device device, void* stream, size_t bytes) {
  THPObjectPtr handle(PyLong_FromVoidPtr(stream));
  if (!handle) throw python_error();
  THPObjectPtr held(PyObject_CallFunction(counters_of, "iOn", (int)device.index(), handle.get(), (Py_ssize_t)bytes));
  if (!held) throw python_error();
  return tensor("counters", held.get());
}

// New codes [R, C], rows at multiples of 16 bytes, and scales of blocks of `block` rows.
struct NewFp8 {
  at::Tensor codes, scales;
  int64_t ld;
  NewFp8(int64_t R, int64_t C, int64_t block, at::ScalarType type, at::Device device) : ld(cdiv(C, 16) * 16) {
    codes = make({R, ld}, type, device);
    if (ld != C) codes = codes.narrow(1, 0, C);
    scales = make({cdiv(R, block), cdiv(C, kGroup)}, at::kFloat, device);
  }
};

PyObject* build_rms(PyObject* const* args) {
  const at::Tensor& x = tensor("x", args[0]);
  OneGpu gpu;
  const int32_t x_code = gpu.code("x", x);
  const Rows r("x", x);
  const Params p(gpu, args[1], Py_None, r.D);
  const bool added = args[2] != Py_None;
  const at::Tensor& res_in = added ? tensor("residual", args[2]) : x;
  const int32_t r_code = gpu.code("residual", res_in);
  if (added && res_in.sizes() != x.sizes()) bad_value("residual has shape " + shape(res_in) + ", x " + shape(x));
  const Rows res("residual", res_in);
  const double eps = number(args[3]);
  const at::ScalarType type = dtype(args[4], x.scalar_type());
  if (!is_wide(type) && !is_fp8(type))
    bad_type(std::string("unsupported dtype ") + toString(type) +
             " (use float32, bfloat16, float8_e4m3fn or float8_e5m2)");
  const c10::DeviceGuard guard(x.device());
  at::Tensor y, y_scale;
  int64_t ldy = r.D;
  if (is_fp8(type)) {
    const NewFp8 q(r.R, r.D, 1, type, x.device());
    y = q.codes, y_scale = q.scales, ldy = q.ld;
  } else {
    y = make(x.sizes(), type, x.device());
  }
  const at::Tensor h = added ? make(x.sizes(), res_in.scalar_type(), x.device()) : x;
  const at::Tensor rstd = make({r.R}, at::kFloat, x.device());
  check(tilec_rms_norm(r.t.const_data_ptr(), added ? res.t.const_data_ptr() : nullptr, data(p.weight), y.data_ptr(),
                       y_scale.defined() ? static_cast<float*>(y_scale.data_ptr()) : nullptr,
                       added ? h.data_ptr() : nullptr, static_cast<float*>(rstd.data_ptr()), r.R, r.D, r.ld, res.ld, ldy,
                       r.D, y_scale.defined() ? y_scale.stride(0) : 0, y_scale.defined() ? y_scale.stride(1) : 0, x_code,
                       r_code, code_of(type), p.code, (float)eps, stream_on(x.device())));
  if (!y_scale.defined()) return tuple({y, h, rstd});
  PyObject* t = PyTuple_New(3);
  if (t == nullptr) throw python_error();
  THPObjectPtr held(t);
  PyTuple_SET_ITEM(t, 0, tuple({y, y_scale}));
  PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(h));
  PyTuple_SET_ITEM(t, 2, THPVariable_Wrap(rstd));
  return held.release();
}

PyObject* build_rms_backward(PyObject* const* args) {
  const at::Tensor &dy = tensor("dy", args[0]), &h = tensor("h", args[1]), &rstd_in = tensor("rstd", args[2]);
  OneGpu gpu;
  const int32_t dy_code = gpu.code("dy", dy), h_code = gpu.code("h", h);
  if (dy.sizes() != h.sizes()) bad_value("dy has shape " + shape(dy) + ", h " + shape(h));
  const Rows d("dy", dy), r("h", h);
  gpu.code("rstd", rstd_in);
  if (rstd_in.scalar_type() != at::kFloat) bad_type("rstd is float32");
  const at::Tensor rstd = vector("rstd", rstd_in, r.R);
  const Params p(gpu, args[3], Py_None, r.D);
  const bool added = args[4] != Py_None;
  const at::Tensor& dh_in = added ? tensor("dh", args[4]) : dy;
  const int32_t dh_code = gpu.code("dh", dh_in);
  if (dh_in.sizes() != h.sizes()) bad_value("dh has shape " + shape(dh_in) + ", h " + shape(h));
  const Rows dh("dh", dh_in);
  const int sums = PyObject_IsTrue(args[5]);
  if (sums < 0) throw python_error();
  const c10::DeviceGuard guard(dy.device());
  const at::Tensor dx = make(dh_in.sizes(), dh_in.scalar_type(), dy.device());
  at::Tensor dw, scratch;
  if (sums) dw = make({r.D}, at::kFloat, dy.device());
  if (sums || r.R > 0) {
    const size_t need = tilec_rms_norm_backward_workspace_bytes(r.R, r.D, h_code);
    if (need > 0) scratch = make({(int64_t)need}, at::kByte, dy.device());
    check(tilec_rms_norm_backward(
        d.t.const_data_ptr(), r.t.const_data_ptr(), static_cast<const float*>(rstd.const_data_ptr()), data(p.weight),
        added ? dh.t.const_data_ptr() : nullptr, dx.data_ptr(), sums ? static_cast<float*>(dw.data_ptr()) : nullptr, r.R,
        r.D, d.ld, r.ld, dh.ld, r.D, dy_code, h_code, dh_code, p.code, need > 0 ? scratch.data_ptr() : nullptr, need,
        stream_on(dy.device())));
  }
  return tuple({dx, dw});
}

// A (codes, scales) pair: codes whose rows are contiguous (copied if they are
// not), scales of blocks of 1 or 128 rows.
struct Fp8 {
  at::Tensor codes, scales;
  int64_t R, C, ld, s_row, s_group;  // strides of the rows of codes and of the scales
  int32_t code, block;
  Fp8(OneGpu& gpu, const char* name, PyObject* o) {
    const std::string of(name);
    if (!PyTuple_Check(o) && !PyList_Check(o)) bad_type(of + " is no pair (codes, scales)");
    const List both(o);
    if (both.size() != 2) bad_value(of + " is no pair (codes, scales)");
    const at::Tensor &c = tensor(name, both[0]), &s = tensor(name, both[1]);
    if (!c.is_cuda() || !s.is_cuda())
      bad_type("needs tensors on a ROCm GPU (" + of + " is on " + (c.is_cuda() ? s : c).device().str() + ")");
    if (gpu.device < 0) gpu.device = c.get_device();
    if (c.get_device() != gpu.device || s.get_device() != gpu.device)
      bad_type("needs all tensors on one GPU (" + of + " is on another)");
    if (c.layout() != at::kStrided || s.layout() != at::kStrided) bad_type(of + " is not a dense tensor");
    if (!is_fp8(c.scalar_type()) || s.scalar_type() != at::kFloat)
      bad_type(of + " has codes of dtype " + toString(c.scalar_type()) + " and scales of dtype " + toString(s.scalar_type()) +
               " (use float8_e4m3fn or float8_e5m2, and float32)");
    if (c.dim() != 2) bad_value("expected 2-D codes of " + of + ", got shape " + shape(c));
    R = c.size(0), C = c.size(1);
    const int64_t G = cdiv(C, kGroup);
    if (s.dim() != 2 || s.size(1) != G || (s.size(0) != R && s.size(0) != cdiv(R, kGroup)))
      bad_value(of + " has codes of shape " + shape(c) + " and scales of shape " + shape(s) + ", expected (" +
                std::to_string(R) + ", " + std::to_string(G) + ") or (" + std::to_string(cdiv(R, kGroup)) + ", " +
                std::to_string(G) + ")");
    block = s.size(0) == R ? 1 : kGroup;
    codes = (C > 1 && c.stride(1) != 1) || (R > 1 && c.stride(0) < C) ? c.contiguous() : c;
    scales = s.size(0) > 1 && s.stride(0) > kMaxScaleRow ? s.contiguous() : s;
    s_row = s.size(0) > 1 ? scales.stride(0) : 0, s_group = G > 1 ? scales.stride(1) : 0;
    ld = R > 1 ? codes.stride(0) : C;
    code = code_of(c.scalar_type());
  }
};

PyObject* build_quantize(PyObject* const* args) {
  const at::Tensor& x = tensor("x", args[0]);
  OneGpu gpu;
  const int32_t x_code = gpu.code("x", x);
  if (x.dim() != 2) bad_value("expected a 2-D x, got shape " + shape(x));
  long long b[2] = {0, 0};
  if (!PyTuple_Check(args[1]) || !PyArg_ParseTuple(args[1], "LL", &b[0], &b[1])) {
    PyErr_Clear();
    bad_value("block is (1, 128) or (128, 128)");
  }
  if ((b[0] != 1 && b[0] != kGroup) || b[1] != kGroup) bad_value("block is (1, 128) or (128, 128)");
  const at::ScalarType type = dtype(args[2], at::kFloat8_e4m3fn);
  if (!is_fp8(type)) bad_type(std::string("unsupported dtype ") + toString(type) + " (use float8_e4m3fn or float8_e5m2)");
  const int64_t R = x.size(0), C = x.size(1);
  at::Tensor t = x;
  const bool rows = (C <= 1 || x.stride(1) == 1) && (R <= 1 || x.stride(0) >= C);
  const bool cols = !rows && (R <= 1 || x.stride(0) == 1) && (C <= 1 || x.stride(1) >= R);
  const c10::DeviceGuard guard(x.device());
  if (!rows && !cols) t = x.contiguous();
  const NewFp8 q(R, C, b[0], type, x.device());
  const int64_t ld = cols ? (C > 1 ? t.stride(1) : R) : (R > 1 ? t.stride(0) : C);
  check(tilec_quantize_fp8(t.const_data_ptr(), q.codes.data_ptr(), static_cast<float*>(q.scales.data_ptr()), R, C, ld,
                           q.ld, q.scales.stride(0), q.scales.stride(1), cols ? TILEC_X1_COL_MAJOR : 0, x_code,
                           code_of(type), (int32_t)b[0], stream_on(x.device())));
  return tuple({q.codes, q.scales});
}

PyObject* build_dequantize(PyObject* const* args) {
  OneGpu gpu;
  const Fp8 q(gpu, "q", args[0]);
  const at::ScalarType type = dtype(args[1], at::kFloat);
  if (!is_wide(type)) bad_type(std::string("unsupported dtype ") + toString(type) + " (use float32 or bfloat16)");
  const c10::DeviceGuard guard(q.codes.device());
  const at::Tensor out = make({q.R, q.C}, type, q.codes.device());
  check(tilec_dequantize_fp8(q.codes.const_data_ptr(), static_cast<const float*>(q.scales.const_data_ptr()),
                             out.data_ptr(),
                             q.R, q.C, q.ld, q.C, q.s_row, q.s_group, q.code, code_of(type), q.block,
                             stream_on(q.codes.device())));
  return THPVariable_Wrap(out);
}

PyObject* build_linear(PyObject* const* args) {
  OneGpu gpu;
  const Fp8 x(gpu, "x", args[0]), w(gpu, "weight", args[1]);
  if (x.C != w.C)
    bad_value("expected x [M, K] and weight [N, K], got shapes " + shape(x.codes) + " and " + shape(w.codes));
  const at::ScalarType type = dtype(args[2], at::kFloat);
  if (!is_wide(type)) bad_type(std::string("unsupported dtype ") + toString(type) + " (use float32 or bfloat16)");
  const c10::DeviceGuard guard(x.codes.device());
  const at::Tensor out = make({x.R, w.R}, type, x.codes.device());
  const void *xp = x.codes.const_data_ptr(), *wp = w.codes.const_data_ptr();
  size_t need = 0, counts = 0;
  check(tilec_linear_fp8_scratch_bytes(xp, wp, x.R, w.R, x.C, x.ld, w.ld, x.code, w.code, code_of(type), &need, &counts));
  void* const stream = stream_on(x.codes.device());
  at::Tensor scratch, counters;
  if (need > 0) scratch = make({(int64_t)need}, at::kByte, x.codes.device());
  if (counts > 0) counters = zeroed(args[3], x.codes.device(), stream, counts);
  check(tilec_linear_fp8(xp, static_cast<const float*>(x.scales.const_data_ptr()), wp,
                         static_cast<const float*>(w.scales.const_data_ptr()), out.data_ptr(), x.R, w.R, x.C, x.ld, w.ld,
                         w.R, x.s_row, x.s_group, w.s_row, w.s_group, x.code, w.code, code_of(type), x.block, w.block,
                         need > 0 ? scratch.data_ptr() : nullptr, need, counts > 0 ? counters.data_ptr() : nullptr,
                         counts, stream));
  return THPVariable_Wrap(out);
}

// The gradients of a list, None for those that have none.  Values whose order in
// memory is another than their index's (a transposed gradient) are as good.
struct Grads {
  std::vector<tilec_grad> table;
  std::vector<at::Tensor> kept;
  Reader r;
  Written w;
  at::Device device = at::kCPU;
  Grads(PyObject* list, bool write) {
    const List grads(list);
    table.reserve(grads.size());
    for (Py_ssize_t i = 0; i < grads.size(); ++i) {
      if (grads[i] == Py_None) continue;
      const at::Tensor* g = &r.read("grads", grads[i], -1, at::kFloat, at::kBFloat16, false);
      device = g->device();
      if (!g->is_non_overlapping_and_dense()) {
        if (write) bad_value("grads has a tensor whose values do not lie side by side");
        kept.push_back(g->contiguous());
        g = &kept.back();
      }
      table.push_back({write ? w.add(*g) : const_cast<void*>(g->const_data_ptr()), g->numel(), code(*g)});
    }
    if (r.device < 0) bad_value("no gradients");
    if (write) refuse_shared();
  }
  // Memory that is multiplied twice would be a race between workgroups.
  void refuse_shared() const {
    std::vector<std::pair<uintptr_t, uintptr_t>> ranges;
    ranges.reserve(table.size());
    for (const tilec_grad& g : table) {
      const uintptr_t lo = reinterpret_cast<uintptr_t>(g.data);
      if (g.n > 0) ranges.emplace_back(lo, lo + (uintptr_t)g.n * (g.dtype == TILEC_BF16 ? 2 : 4));
    }
    std::sort(ranges.begin(), ranges.end());
    for (size_t i = 1; i < ranges.size(); ++i)
      if (ranges[i].first < ranges[i - 1].second) bad_value("two grads share their memory");
  }
};

// Enqueues the norm; {norm, scale}.  args: grads, max_norm, grad_scale, counters_of.
std::pair<at::Tensor, at::Tensor> norm_of(Grads& g, PyObject* const* args, void*& stream) {
  const double max_norm = args[1] == Py_None ? -1. : number(args[1]);
  if (args[1] != Py_None && !(max_norm >= 0)) bad_value("max_norm is negative or not a number");
  const float* grad_scale = nullptr;
  if (args[2] != Py_None) {
    const at::Tensor& t = g.r.read("grad_scale", args[2], -1, at::kFloat, at::kFloat, false);
    if (t.numel() != 1) bad_value("grad_scale has shape " + shape(t) + ", expected one value");
    grad_scale = static_cast<const float*>(t.const_data_ptr());
  }
  stream = stream_on(g.device);
  const at::Tensor counter = zeroed(args[3], g.device, stream, sizeof(unsigned));
  const at::Tensor norm = make({}, at::kFloat, g.device), scale = make({}, at::kFloat, g.device);
  const size_t need = tilec_grad_norm_workspace_bytes(g.table.data(), (int32_t)g.table.size());
  at::Tensor scratch;
  if (need > 0) scratch = make({(int64_t)need}, at::kByte, g.device);
  check(tilec_grad_norm(g.table.data(), (int32_t)g.table.size(), grad_scale, max_norm,
                        static_cast<float*>(norm.data_ptr()), static_cast<float*>(scale.data_ptr()),
                        need > 0 ? scratch.data_ptr() : nullptr, need, counter.data_ptr(), (size_t)counter.numel(), stream));
  return {norm, scale};
}

PyObject* build_grad_norm(PyObject* const* args) {
  Grads g(args[0], false);
  const c10::DeviceGuard guard(g.device);
  void* stream;
  const auto got = norm_of(g, args, stream);
  return tuple({got.first, got.second});
}

PyObject* build_clip(PyObject* const* args) {
  Grads g(args[0], true);
  const c10::DeviceGuard guard(g.device);
  void* stream;
  const auto got = norm_of(g, args, stream);
  check(tilec_scale_grads(g.table.data(), (int32_t)g.table.size(), static_cast<const float*>(got.second.const_data_ptr()),
                          stream));
  g.w.bump();
  return THPVariable_Wrap(got.first);
}

constexpr char kAdamw[] = "adamw_step", kValues[] = "adamw_values", kNorm[] = "layer_norm", kNormBackward[] = "layer_norm_backward";
constexpr char kRms[] = "rms_norm", kRmsBackward[] = "rms_norm_backward", kQuantize[] = "quantize_fp8",
               kDequantize[] = "dequantize_fp8", kLinear[] = "linear_fp8", kGradNorm[] = "grad_norm", kClip[] = "clip_grads";

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
    {"rms_norm", function<build_rms, 5, kRms>(), METH_FASTCALL,
     "rms_norm(x, weight, residual, eps, dtype) -> (y, h, rstd)"},
    {"rms_norm_backward", function<build_rms_backward, 6, kRmsBackward>(), METH_FASTCALL,
     "rms_norm_backward(dy, h, rstd, weight, dh, weight_grad) -> (dx, dweight)"},
    {"quantize_fp8", function<build_quantize, 3, kQuantize>(), METH_FASTCALL,
     "quantize_fp8(x, block, dtype) -> (codes, scales)"},
    {"dequantize_fp8", function<build_dequantize, 2, kDequantize>(), METH_FASTCALL,
     "dequantize_fp8(q, dtype) -> values"},
    {"linear_fp8", function<build_linear, 4, kLinear>(), METH_FASTCALL,
     "linear_fp8(x, weight, dtype, counters_of) -> out"},
    {"grad_norm", function<build_grad_norm, 4, kGradNorm>(), METH_FASTCALL,
     "grad_norm(grads, max_norm, grad_scale, counters_of) -> (norm, scale)"},
    {"clip_grads", function<build_clip, 4, kClip>(), METH_FASTCALL,
     "clip_grads(grads, max_norm, grad_scale, counters_of) -> norm"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&kModule); }
