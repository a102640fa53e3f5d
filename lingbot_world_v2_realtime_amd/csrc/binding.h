// What the bindings of the block operators and of causal attention share: checks of arguments, errors, and the rotation's
// arguments. Every function takes its arguments by position (kernels.py and layers/ hold the signatures that users see),
// runs on the current stream of its first tensor's device, with that device current, and raises ValueError / TypeError for
// what it does not take. A status from the library goes to the function that `on_status` was given, which raises.
#pragma once

#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include <algorithm>
#include <array>
#include <optional>
#include <sstream>
#include <string>

#include "lbw_attn.h"
#include "lbw_block.h"
#include "lbw_causal.h"

namespace lbw_py {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Maybe = std::optional<Tensor>;

inline PyObject* status_handler = nullptr;

template <typename... A>
inline std::string text(const A&... a) {
  std::ostringstream s;
  (s << ... << a);
  return s.str();
}
template <typename... A>
[[noreturn]] inline void value_error(const A&... a) {
  PyErr_SetString(PyExc_ValueError, text(a...).c_str());
  throw python_error();
}
template <typename... A>
[[noreturn]] inline void type_error(const A&... a) {
  PyErr_SetString(PyExc_TypeError, text(a...).c_str());
  throw python_error();
}

inline std::string dims(at::IntArrayRef v) {
  std::string s = "(";
  for (size_t i = 0; i < v.size(); ++i) s += (i ? ", " : "") + std::to_string(v[i]);
  return s + (v.size() == 1 ? ",)" : ")");
}

inline const Tensor absent;

inline const Tensor& tensor(const char* name, PyObject* o, bool optional = false) {
  if (optional && o == Py_None) return absent;
  if (!THPVariable_Check(o)) type_error(name, " must be a tensor, got ", Py_TYPE(o)->tp_name);
  const Tensor& t = THPVariable_Unpack(o);
  if (t.is_neg()) value_error(name, " is a lazily negated view: give its resolve_neg()");
  // (an address of zero means that the tensor is absent)
  if (t.numel() && !t.const_data_ptr()) type_error(name, " has no memory of its own, got ", Py_TYPE(o)->tp_name);
  return t;
}

inline double number(const char* name, PyObject* o) {
  if (THPVariable_Check(o)) type_error(name, " must be a number, got a tensor (whose gradient would be lost)");
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    type_error(name, " must be a number, got ", Py_TYPE(o)->tp_name);
  }
  return v;
}

inline int64_t integer(const char* name, PyObject* o) {
  PyObject* i = PyNumber_Index(o);
  if (!i) {
    PyErr_Clear();
    type_error(name, " must be an integer, got ", Py_TYPE(o)->tp_name);
  }
  int overflow = 0;
  const int64_t v = PyLong_AsLongLongAndOverflow(i, &overflow);
  Py_DECREF(i);
  if (overflow) value_error(name, " is out of range");
  return v;
}

inline bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw python_error();
  return v;
}

inline std::string word(const char* name, PyObject* o) {
  if (!PyUnicode_Check(o)) type_error(name, " must be a string, got ", Py_TYPE(o)->tp_name);
  const char* s = PyUnicode_AsUTF8(o);
  if (!s) throw python_error();
  return s;
}

inline int element_format(const char* name, const Tensor& t) {
  const auto d = t.scalar_type();
  const int code = d == at::kBFloat16 ? LBW_DTYPE_BF16 : d == at::kHalf ? LBW_DTYPE_FP16 : d == at::kFloat ? LBW_DTYPE_FP32 : -1;
  if (code < 0) type_error(name, " must be bfloat16, float16 or float32, got ", d);
  return code;
}

inline void on_device(const char* name, const Tensor& t) {
  if (!t.is_cuda()) value_error(name, " must be a device tensor (the block operators have no CPU implementation)");
}

inline int row_format(const char* name, const Tensor& t) {
  const int code = element_format(name, t);
  on_device(name, t);
  return code;
}

inline bool unit_stride(const Tensor& t) { return t.dim() >= 1 && (t.size(-1) <= 1 || t.stride(-1) == 1); }

template <typename... T>
inline void same_device(const char* what, const Tensor& first, const T&... rest) {
  const auto check = [&](const Tensor& t) {
    if (t.defined() && t.device() != first.device())
      value_error(what, ": tensors on different devices ", first.device(), " and ", t.device());
  };
  (check(rest), ...);
}

// (a gradient that a hook replaced by a tensor without memory must not count as absent either)
inline void* ptr(const Tensor& t) {
  if (!t.defined()) return nullptr;
  void* p = t.data_ptr();
  TORCH_CHECK(p || !t.numel(), "a tensor without memory of its own");
  return p;
}

// The device of a call made current, and its current stream.
struct On {
  c10::hip::HIPGuard guard;
  void* stream;
  explicit On(const Tensor& t) : guard(t.device().index()), stream(c10::hip::getCurrentHIPStream(t.device().index()).stream()) {}
};

// A bad status: raised by the Python side's function, or, in a backward pass (which runs without the interpreter), as
// torch's error.
inline void done(int status, const char* what, bool python = true) {
  if (status == LBW_OK) return;
  TORCH_CHECK(python, what, " failed: status ", status, " (", lbw_status_string(status), ")");
  PyObject* r = status_handler ? PyObject_CallFunction(status_handler, "is", status, what) : nullptr;
  Py_XDECREF(r);
  if (PyErr_Occurred()) throw python_error();
  value_error(what, " failed: status ", status);
}

inline Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : std::nullopt; }

// Whether autograd has to see the call: a gradient is recorded, or an input carries a forward-mode tangent (which it
// refuses).
inline bool records_gradient(const Tensor& t) {
  if (!t.defined() || !t.unsafeGetTensorImpl()->autograd_meta()) return false;   // (a plain tensor has none)
  return (c10::GradMode::is_enabled() && t.requires_grad()) || t._fw_grad(0).defined();
}
template <typename... T>
inline bool records_gradient(const Tensor& t, const T&... rest) {
  return records_gradient(t) || records_gradient(rest...);
}

// For the calls that have no gradient of their own: a tensor that would record one is refused (the result would be
// detached).
inline void no_gradient(const char* what, bool recorded) {
  if (!recorded) return;
  PyErr_Format(PyExc_RuntimeError, "%s records no gradient: call it under torch.no_grad(), or on detached tensors", what);
  throw python_error();
}
inline void no_gradient(const char* what, PyObject* const* args, Py_ssize_t n) {   // (before anything else looks at them)
  for (Py_ssize_t i = 0; i < n; ++i)
    if (args[i] != Py_None && THPVariable_Check(args[i])) no_gradient(what, records_gradient(THPVariable_Unpack(args[i])));
}

inline Tensor new_like(const Tensor& t) { return at::empty(t.sizes(), t.options()); }   // (packed, whatever t's strides)

inline PyObject* wrap(const Tensor& t) {
  if (!t.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(t);
}

template <size_t N>
inline PyObject* wrap_all(const std::array<Tensor, N>& ts) {
  PyObject* out = PyTuple_New(N);
  if (!out) throw python_error();
  for (size_t i = 0; i < N; ++i) PyTuple_SET_ITEM(out, i, wrap(ts[i]));
  return out;
}

inline void count(Py_ssize_t got, Py_ssize_t want) {
  if (got != want) type_error("expected ", want, " arguments, got ", got);
}

struct RotaryOptions : torch::CustomClassHolder {
  int64_t start = 0;
  double factor = 1.0;
  bool interleaved = true, nhd = true;
};

struct Rotary {
  Tensor q, k, pos, freq, axis;
  c10::intrusive_ptr<RotaryOptions> o;

  Rotary() = default;
  // q, k, positions, freq, axis, pairs, factor, layout, axes, checked (but for the device: that comes last, so that
  // every other refusal can be seen without one)
  explicit Rotary(PyObject* const* args)
      : q(tensor("q", args[0])), k(tensor("k", args[1], true)), freq(tensor("freq", args[3])), axis(tensor("axis", args[4], true)),
        o(c10::make_intrusive<RotaryOptions>()) {
    element_format("q", q);
    const std::string layout = word("layout", args[7]), pairs = word("pairs", args[5]);
    if (layout != "NHD" && layout != "HND") value_error("tensor_layout must be 'NHD' or 'HND', got '", layout, "'");
    o->nhd = layout == "NHD";
    if (pairs != "interleaved" && pairs != "half") value_error("pairs must be 'interleaved' or 'half', got '", pairs, "'");
    o->interleaved = pairs == "interleaved";
    o->factor = number("factor", args[6]);
    for (const Tensor* t : {&q, &k}) {
      if (!t->defined()) continue;
      if (t->dim() != 4) value_error("expected a 4-d tensor, got shape ", dims(t->sizes()));
      if (!unit_stride(*t)) value_error("q and k must have contiguous channels");
    }
    const int64_t b = q.size(0), len = q.size(tok()), d = q.size(3);
    if (k.defined()) {
      if (k.scalar_type() != q.scalar_type())
        type_error("q (", q.scalar_type(), ") and k (", k.scalar_type(), ") must have one dtype");
      if (k.size(0) != b || k.size(tok()) != len || k.size(3) != d)
        value_error("q ", dims(q.sizes()), " and k ", dims(k.sizes()), " do not match");
    }
    if (q.numel() + (k.defined() ? k.numel() : 0) > 0 && (q.size(head()) < 1 || (k.defined() && k.size(head()) < 1)))
      value_error("q and k need a head at least");
    if (freq.scalar_type() != at::kDouble || freq.dim() != 1 || !freq.is_contiguous() || freq.size(0) < 1)
      value_error("freq must be contiguous float64 [pairs], got ", freq.scalar_type(), " ", dims(freq.sizes()));
    if (records_gradient(freq)) value_error("freq has no gradient: detach it");
    if (2 * freq.size(0) > d || d > LBW_ROTARY_MAX_DIM)
      value_error(freq.size(0), " pairs do not fit heads of ", d, " (of ", LBW_ROTARY_MAX_DIM, " at most)");
    if (axis.defined() && (axis.scalar_type() != at::kInt || axis.sizes() != freq.sizes() || !axis.is_contiguous()))
      value_error("axis must be contiguous int32 ", dims(freq.sizes()), ", got ", axis.scalar_type(), " ", dims(axis.sizes()));
    const int64_t axes = args[8] == Py_None ? 1 : integer("axes", args[8]);   // (None: not known here)
    if (axes < 1 || (axes > 1 && !axis.defined()))
      value_error("a plan of ", axes, " axes", axes > 1 ? " needs the axis of each pair" : "");
    if (THPVariable_Check(args[2])) {
      pos = tensor("positions", args[2]);
      if (pos.scalar_type() != at::kInt && pos.scalar_type() != at::kLong)
        type_error("positions must be int32 or int64, got ", pos.scalar_type());
      const int64_t own = own_dims();
      if (!((own == 1 && pos.size(0) == len) || (own == 2 && pos.size(0) == b && pos.size(1) == len)))
        value_error("positions must be [", len, "] or [", b, ", ", len, "]", axis.defined() ? " x axes" : "", ", got ",
                    dims(pos.sizes()));
      if (axis.defined() && pos.size(own) < axes)
        value_error("positions ", dims(pos.sizes()), " have ", pos.size(own), " axes, the plan has ", axes, " axes");
    } else {
      if (axis.defined()) value_error("several axes need a positions tensor");
      o->start = integer("positions", args[2]);
    }
    same_device("rotary", q, k, pos, freq, axis);
  }
  int tok() const { return o->nhd ? 1 : 2; }
  int head() const { return o->nhd ? 2 : 1; }
  int64_t own_dims() const { return pos.dim() - (axis.defined() ? 1 : 0); }   // of positions, without an axis dimension behind

  void run(const Tensor& qo, const Tensor& ko, bool inverse, bool python) const {
    if (python) on_device("q", q);
    if (q.numel() + (k.defined() ? k.numel() : 0) == 0) return;
    const int64_t own = pos.defined() ? own_dims() : 0;
    const auto st = [&](const Tensor& t, int dim) { return t.defined() ? t.stride(dim) : 0; };
    const On on(q);
    done(lbw_rotary(q.data_ptr(), ptr(k), element_format("q", q), q.size(0), q.size(tok()), q.size(head()),
                    k.defined() ? k.size(head()) : 0, q.size(3), freq.size(0), st(q, 0), st(q, tok()), st(q, head()), st(k, 0),
                    st(k, tok()), st(k, head()), ptr(pos), pos.defined() && pos.scalar_type() == at::kLong,
                    own == 2 ? pos.stride(0) : 0, own ? pos.stride(own - 1) : 0, own && axis.defined() ? pos.stride(own) : 0,
                    o->start, (const double*)freq.data_ptr(), (const int32_t*)ptr(axis),
                    own && axis.defined() ? pos.size(own) : 1, o->interleaved, inverse, (float)o->factor, qo.data_ptr(), ptr(ko),
                    st(qo, 0), st(qo, tok()), st(qo, head()), st(ko, 0), st(ko, tok()), st(ko, head()), on.stream),
         "lbw_rotary", python);
  }
  // into new tensors
  std::array<Tensor, 2> fresh(bool inverse, bool python) const {
    const std::array<Tensor, 2> out = {new_like(q), k.defined() ? new_like(k) : Tensor()};
    run(out[0], out[1], inverse, python);
    return out;
  }
};

// causal_binding.cpp
PyObject* norm_rotary_embed(PyObject*, PyObject* const*, Py_ssize_t);
PyObject* packed_attention(PyObject*, PyObject* const*, Py_ssize_t);
PyObject* kv4_write(PyObject*, PyObject* const*, Py_ssize_t);
PyObject* kv4_read(PyObject*, PyObject* const*, Py_ssize_t);
PyObject* kv4_attend(PyObject*, PyObject* const*, Py_ssize_t);

}  // namespace lbw_py
