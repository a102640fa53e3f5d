// The block operators' calls from Python: tensors checked, outputs allocated and the C-ABI of include/lbw_block.h called in
// one native step. A call of these is bound by its host side (a token's norm takes 4 us on the GPU); the same checks and the
// 33 arguments of a ctypes call took 15-19 us in Python, against 5 here.
//
// Every function takes its arguments by position (kernels.py holds the signatures that users see), runs on the current
// stream of its first tensor's device, with that device current, and raises ValueError / TypeError for what it does not
// take. A status from the library goes to the function that `on_status` was given, which raises.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <array>
#include <sstream>
#include <string>

#include "lbw_attn.h"
#include "lbw_block.h"

namespace {

using at::Tensor;

PyObject* status_handler = nullptr;

template <typename... A>
std::string text(const A&... a) {
  std::ostringstream s;
  (s << ... << a);
  return s.str();
}
template <typename... A>
[[noreturn]] void value_error(const A&... a) {
  PyErr_SetString(PyExc_ValueError, text(a...).c_str());
  throw python_error();
}
template <typename... A>
[[noreturn]] void type_error(const A&... a) {
  PyErr_SetString(PyExc_TypeError, text(a...).c_str());
  throw python_error();
}

std::string dims(at::IntArrayRef v) {
  std::string s = "(";
  for (size_t i = 0; i < v.size(); ++i) s += (i ? ", " : "") + std::to_string(v[i]);
  return s + (v.size() == 1 ? ",)" : ")");
}

const Tensor absent;

const Tensor& tensor(const char* name, PyObject* o, bool optional = false) {
  if (optional && o == Py_None) return absent;
  if (!THPVariable_Check(o)) type_error(name, " must be a tensor, got ", Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}

double number(const char* name, PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    type_error(name, " must be a number, got ", Py_TYPE(o)->tp_name);
  }
  return v;
}

int64_t integer(const char* name, PyObject* o) {
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

std::string word(const char* name, PyObject* o) {
  if (!PyUnicode_Check(o)) type_error(name, " must be a string, got ", Py_TYPE(o)->tp_name);
  const char* s = PyUnicode_AsUTF8(o);
  if (!s) throw python_error();
  return s;
}

int row_format(const char* name, const Tensor& t) {
  const auto d = t.scalar_type();
  const int code = d == at::kBFloat16 ? LBW_DTYPE_BF16 : d == at::kHalf ? LBW_DTYPE_FP16 : d == at::kFloat ? LBW_DTYPE_FP32 : -1;
  if (code < 0) type_error(name, " must be bfloat16, float16 or float32, got ", d);
  if (!t.is_cuda()) value_error(name, " must be a device tensor (the block operators have no CPU implementation)");
  return code;
}

bool unit_stride(const Tensor& t) { return t.dim() >= 1 && (t.size(-1) <= 1 || t.stride(-1) == 1); }

template <typename... T>
void same_device(const char* what, const Tensor& first, const T&... rest) {
  const auto check = [&](const Tensor& t) {
    if (t.defined() && t.device() != first.device())
      value_error(what, ": tensors on different devices ", first.device(), " and ", t.device());
  };
  (check(rest), ...);
}

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// The device of a call made current, and its current stream.
struct On {
  c10::hip::HIPGuard guard;
  void* stream;
  explicit On(const Tensor& t) : guard(t.device().index()), stream(c10::hip::getCurrentHIPStream(t.device().index()).stream()) {}
};

void done(int status, const char* what) {
  if (status == LBW_OK) return;
  PyObject* r = status_handler ? PyObject_CallFunction(status_handler, "is", status, what) : nullptr;
  Py_XDECREF(r);
  if (PyErr_Occurred()) throw python_error();
  value_error(what, " failed: status ", status);
}

Tensor new_like(const Tensor& t) { return at::empty(t.sizes(), t.options()); }   // (packed, whatever t's strides)

PyObject* wrap(const Tensor& t) {
  if (!t.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(t);
}

template <size_t N>
PyObject* wrap_all(const std::array<Tensor, N>& ts) {
  PyObject* out = PyTuple_New(N);
  if (!out) throw python_error();
  for (size_t i = 0; i < N; ++i) PyTuple_SET_ITEM(out, i, wrap(ts[i]));
  return out;
}

void count(Py_ssize_t got, Py_ssize_t want) {
  if (got != want) type_error("expected ", want, " arguments, got ", got);
}

// ---------------------------------------------------------------- gated norm

enum { GATE, SHIFT, SCALE, WEIGHT, BIAS, POST_WEIGHT, VECTORS };
const char* const VECTOR_NAMES[VECTORS] = {"gate", "shift", "scale", "weight", "bias", "post_weight"};

int norm_kind(const char* name, PyObject* o) {
  if (o == Py_None) return LBW_NORM_NONE;
  const std::string s = PyUnicode_Check(o) ? word(name, o) : "";
  if (s == "layer") return LBW_NORM_LAYER;
  if (s == "rms") return LBW_NORM_RMS;
  value_error(name, " must be 'layer', 'rms' or None");
}

// The arguments of a norm and of its gradient: x, y, the vectors, norm, post_norm, eps, residual_scale, branch_scale, group_len.
struct Norm {
  static constexpr int ARGS = 2 + VECTORS + 6;
  const Tensor &x, &y;
  const Tensor* v[VECTORS];
  int norm, post, dtype, vec_dtype;
  float eps, a, b;
  int64_t batch, len, width, groups = 1, group_len;
  int rowwise = 0;

  explicit Norm(PyObject* const* o) : x(tensor("x", o[0])), y(tensor("y", o[1], true)) {
    for (int i = 0; i < VECTORS; ++i) v[i] = &tensor(VECTOR_NAMES[i], o[2 + i], true);
    o += 2 + VECTORS;
    dtype = vec_dtype = row_format("x", x);
    if (x.dim() != 3 || !unit_stride(x) || x.size(2) < 1 || x.size(2) > LBW_NORM_MAX_WIDTH)
      value_error("x must be [B, L, C] with contiguous channels, C up to ", LBW_NORM_MAX_WIDTH, ", got ", dims(x.sizes()), " / ",
                  dims(x.strides()));
    batch = x.size(0), len = x.size(1), width = x.size(2);
    norm = norm_kind("norm", o[0]), post = norm_kind("post_norm", o[1]);
    eps = (float)number("eps", o[2]), a = (float)number("residual_scale", o[3]), b = (float)number("branch_scale", o[4]);
    if (y.defined()) {
      if (y.scalar_type() != x.scalar_type()) type_error("x (", x.scalar_type(), ") and y (", y.scalar_type(), ") must have one dtype");
      if (y.sizes() != x.sizes() || !unit_stride(y))
        value_error("y ", dims(y.sizes()), " / ", dims(y.strides()), " must be ", dims(x.sizes()), " with contiguous channels");
    } else if (post || v[GATE]->defined() || v[POST_WEIGHT]->defined()) {
      value_error("gate, post_norm and post_weight act on the branch: give y");
    }
    if (!norm) {
      for (int i : {WEIGHT, BIAS, SHIFT, SCALE})
        if (v[i]->defined()) value_error("weight, bias, shift and scale follow the norm: give one");
      if (!y.defined()) value_error("nothing to do: give y or a norm");
    }
    same_device("gated_norm", x, y, *v[0], *v[1], *v[2], *v[3], *v[4], *v[5]);
    const Tensor* first = nullptr;
    int64_t rows = -1;
    for (int i = 0; i < VECTORS; ++i) {
      const Tensor& t = *v[i];
      if (!t.defined()) continue;
      const auto d = t.scalar_type();
      if ((d != x.scalar_type() && d != at::kFloat) || (first && d != first->scalar_type()))
        type_error("the vectors must all be ", x.scalar_type(), " or all float32, got ", VECTOR_NAMES[i], " of ", d);
      first = &t;
      const bool many = i <= SCALE && t.dim() == 3;
      if (!unit_stride(t) || !(many ? t.size(0) == batch && t.size(2) == width : t.dim() == 1 && t.size(0) == width))
        value_error(VECTOR_NAMES[i], " must be [", width, "]", i <= SCALE ? text(" or [", batch, ", rows, ", width, "]") : "",
                    " with contiguous channels, got ", dims(t.sizes()), " / ", dims(t.strides()));
      if (!many) continue;
      rowwise |= 1 << i;
      if (rows >= 0 && rows != t.size(1)) value_error("modulation vectors with ", rows, " and ", t.size(1), " rows");
      rows = t.size(1);
    }
    if (first) vec_dtype = row_format("vectors", *first);
    group_len = o[5] == Py_None ? 0 : integer("group_len", o[5]);
    if (rows < 0) {
      if (o[5] != Py_None) value_error("group_len is for modulation vectors with rows ([B, rows, C])");
      group_len = len > 0 ? len : 1;
      return;
    }
    if (rows < 1) value_error("modulation vectors need a row at least");
    groups = rows;
    if (o[5] == Py_None) group_len = std::max<int64_t>((len + rows - 1) / rows, 1);
    // (a row may hold more tokens than there are: no overflow in the product)
    if (group_len < 1 || (len + group_len - 1) / group_len > rows || group_len > (1 << 30))
      value_error(rows, " modulation rows of ", group_len, " tokens do not cover ", len, " tokens");
  }
  int64_t stride(int i, int dim) const { return rowwise >> i & 1 ? v[i]->stride(dim) : 0; }
  bool empty() const { return batch * len == 0; }
};

PyObject* gated_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, Norm::ARGS + 1);
  const Norm a(args);
  const bool want_stream = args[Norm::ARGS] == Py_True || !a.norm;
  Tensor s = want_stream ? new_like(a.x) : Tensor(), h = a.norm ? new_like(a.x) : Tensor();
  if (!a.empty()) {
    const On on(a.x);
    done(lbw_gated_norm(a.x.data_ptr(), ptr(a.y), a.dtype, a.vec_dtype, a.batch, a.len, a.width, a.x.stride(0), a.x.stride(1),
                        a.y.defined() ? a.y.stride(0) : 0, a.y.defined() ? a.y.stride(1) : 0, ptr(*a.v[GATE]), a.stride(GATE, 0),
                        a.stride(GATE, 1), ptr(*a.v[SHIFT]), a.stride(SHIFT, 0), a.stride(SHIFT, 1), ptr(*a.v[SCALE]),
                        a.stride(SCALE, 0), a.stride(SCALE, 1), a.group_len, ptr(*a.v[WEIGHT]), ptr(*a.v[BIAS]),
                        ptr(*a.v[POST_WEIGHT]), a.norm, a.post, a.eps, a.a, a.b, ptr(s), ptr(h), on.stream),
         "lbw_gated_norm");
  }
  return wrap_all(std::array<Tensor, 2>{s, h});
  END_HANDLE_TH_ERRORS
}

// After the norm's arguments: ds, dh, and which of x, y and the vectors want a gradient (a bit each). A tuple of those, None
// for the others.
PyObject* gated_norm_bwd(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, Norm::ARGS + 3);
  const Norm a(args);
  const Tensor &ds = tensor("ds", args[Norm::ARGS], true), &dh = tensor("dh", args[Norm::ARGS + 1], true);
  const int64_t wants = integer("wants", args[Norm::ARGS + 2]);
  for (const auto& [name, d] : {std::pair<const char*, const Tensor&>{"ds", ds}, {"dh", dh}})
    if (d.defined() && (d.scalar_type() != a.x.scalar_type() || d.sizes() != a.x.sizes() || !d.is_contiguous()))
      value_error(name, " must be contiguous ", a.x.scalar_type(), " ", dims(a.x.sizes()), ", got ", d.scalar_type(), " ",
                  dims(d.sizes()));
  if (dh.defined() && !a.norm) value_error("dh without a norm");
  same_device("gated_norm_bwd", a.x, ds, dh);
  std::array<Tensor, 2 + VECTORS> g;
  void* p[2 + VECTORS] = {};
  bool sums = false;
  const bool none = (!ds.defined() && !dh.defined()) || a.empty();
  for (int i = 0; i < 2 + VECTORS; ++i) {
    const Tensor& t = i == 0 ? a.x : i == 1 ? a.y : *a.v[i - 2];
    if (!(wants >> i & 1) || !t.defined()) continue;
    // what only the norm's output depends on has a gradient of zero without dh
    const bool idle = none || (!dh.defined() && i >= 2 + SHIFT && i <= 2 + BIAS);
    g[i] = idle ? at::zeros(t.sizes(), t.options()) : new_like(t);
    if (idle) continue;
    p[i] = g[i].data_ptr();
    sums = sums || i >= 2;
  }
  if (!none) {
    const On on(a.x);
    Tensor ws;
    if (sums)
      ws = at::empty({lbw_gated_norm_bwd_workspace_bytes(a.batch, a.len, a.width, a.groups, a.group_len)},
                     a.x.options().dtype(at::kByte));
    done(lbw_gated_norm_bwd(ptr(ds), ptr(dh), a.x.data_ptr(), ptr(a.y), a.dtype, a.vec_dtype, a.batch, a.len, a.width, a.x.stride(0),
                            a.x.stride(1), a.y.defined() ? a.y.stride(0) : 0, a.y.defined() ? a.y.stride(1) : 0, ptr(*a.v[GATE]),
                            a.stride(GATE, 0), a.stride(GATE, 1), ptr(*a.v[SCALE]), a.stride(SCALE, 0), a.stride(SCALE, 1),
                            a.rowwise, a.groups, a.group_len, ptr(*a.v[WEIGHT]), ptr(*a.v[BIAS]), ptr(*a.v[POST_WEIGHT]), a.norm,
                            a.post, a.eps, a.a, a.b, p[0], p[1], p[2 + GATE], p[2 + SHIFT], p[2 + SCALE], p[2 + WEIGHT],
                            p[2 + BIAS], p[2 + POST_WEIGHT], ptr(ws), on.stream),
         "lbw_gated_norm_bwd");
  }
  return wrap_all(g);
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------- rotary

// q, k, positions, freq, axis, pairs, factor, layout, inverse, q_out, k_out
PyObject* rotary(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 11);
  const Tensor &q = tensor("q", args[0]), &k = tensor("k", args[1], true);
  const Tensor &freq = tensor("freq", args[3]), &axis = tensor("axis", args[4], true);
  const int dtype = row_format("q", q);
  const std::string layout = word("layout", args[7]), pairs = word("pairs", args[5]);
  if (layout != "NHD" && layout != "HND") value_error("tensor_layout must be 'NHD' or 'HND', got '", layout, "'");
  const int tok = layout == "NHD" ? 1 : 2, head = 3 - tok;
  for (const Tensor* t : {&q, &k}) {
    if (!t->defined()) continue;
    if (t->dim() != 4) value_error("expected a 4-d tensor, got shape ", dims(t->sizes()));
    if (!unit_stride(*t)) value_error("q and k must have contiguous channels");
  }
  const int64_t b = q.size(0), len = q.size(tok), d = q.size(3);
  if (k.defined()) {
    if (k.scalar_type() != q.scalar_type()) type_error("q (", q.scalar_type(), ") and k (", k.scalar_type(), ") must have one dtype");
    if (k.size(0) != b || k.size(tok) != len || k.size(3) != d)
      value_error("q ", dims(q.sizes()), " and k ", dims(k.sizes()), " do not match");
  }
  if (pairs != "interleaved" && pairs != "half") value_error("pairs must be 'interleaved' or 'half', got '", pairs, "'");
  if (freq.scalar_type() != at::kDouble || freq.dim() != 1 || !freq.is_contiguous() || freq.size(0) < 1)
    value_error("freq must be contiguous float64 [pairs], got ", freq.scalar_type(), " ", dims(freq.sizes()));
  if (2 * freq.size(0) > d || d > LBW_ROTARY_MAX_DIM)
    value_error(freq.size(0), " pairs do not fit heads of ", d, " (of ", LBW_ROTARY_MAX_DIM, " at most)");
  if (axis.defined() && (axis.scalar_type() != at::kInt || axis.sizes() != freq.sizes() || !axis.is_contiguous()))
    value_error("axis must be contiguous int32 ", dims(freq.sizes()), ", got ", axis.scalar_type(), " ", dims(axis.sizes()));
  const bool given = THPVariable_Check(args[2]);
  const Tensor& pos = given ? tensor("positions", args[2]) : absent;
  int64_t ps[3] = {0, 0, 0}, start = 0, axes = 1;
  if (given) {
    if (pos.scalar_type() != at::kInt && pos.scalar_type() != at::kLong)
      type_error("positions must be int32 or int64, got ", pos.scalar_type());
    const int64_t own = pos.dim() - (axis.defined() ? 1 : 0);   // [L] or [B, L], with an axis dimension behind
    if (!((own == 1 && pos.size(0) == len) || (own == 2 && pos.size(0) == b && pos.size(1) == len)))
      value_error("positions must be [", len, "] or [", b, ", ", len, "]", axis.defined() ? " x axes" : "", ", got ", dims(pos.sizes()));
    ps[0] = own == 2 ? pos.stride(0) : 0;
    ps[1] = pos.stride(own - 1);
    if (axis.defined()) {
      ps[2] = pos.stride(own);
      axes = pos.size(own);
      if (axes < 1) value_error("positions need an axis at least");
    }
  } else {
    if (axis.defined()) value_error("several axes need a positions tensor");
    start = integer("positions", args[2]);
  }
  std::array<Tensor, 2> out;
  for (int i = 0; i < 2; ++i) {
    const Tensor &x = i ? k : q, &o = tensor(i ? "k_out" : "q_out", args[9 + i], true);
    const char* name = i ? "k_out" : "q_out";
    if (!x.defined()) {
      if (o.defined()) value_error("k_out without k");
      continue;
    }
    out[i] = o.defined() ? o : new_like(x);
    if (!o.defined()) continue;
    if (o.scalar_type() != x.scalar_type() || o.sizes() != x.sizes() || !unit_stride(o))
      value_error(name, " must be ", x.scalar_type(), " ", dims(x.sizes()), " with contiguous channels");
    for (int j = 0; j < 4; ++j)
      if (o.stride(j) == 0 && o.size(j) > 1) value_error(name, " has elements that share their memory");
    if (o.numel() && o.data_ptr() == x.data_ptr() && o.strides() != x.strides())
      value_error(name, " overlaps its input in another order");
  }
  same_device("rotary", q, k, pos, freq, axis, out[0], out[1]);
  if (q.numel() + (k.defined() ? k.numel() : 0) > 0) {
    if (q.size(head) < 1 || (k.defined() && k.size(head) < 1)) value_error("q and k need a head at least");
    const On on(q);
    const auto st = [&](const Tensor& t, int dim) { return t.defined() ? t.stride(dim) : 0; };
    done(lbw_rotary(q.data_ptr(), ptr(k), dtype, b, len, q.size(head), k.defined() ? k.size(head) : 0, d, freq.size(0), st(q, 0),
                    st(q, tok), st(q, head), st(k, 0), st(k, tok), st(k, head), ptr(pos), given && pos.scalar_type() == at::kLong,
                    ps[0], ps[1], ps[2], start, (const double*)freq.data_ptr(), (const int32_t*)ptr(axis), axes,
                    pairs == "interleaved", PyObject_IsTrue(args[8]), (float)number("factor", args[6]), out[0].data_ptr(),
                    ptr(out[1]), st(out[0], 0), st(out[0], tok), st(out[0], head), st(out[1], 0), st(out[1], tok),
                    st(out[1], head), on.stream),
         "lbw_rotary");
  }
  return wrap_all(out);
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------- 4-bit linears

// x, w4, scale, zero, bias, out_features, fmt
PyObject* gemm_w4(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  count(n_args, 7);
  const Tensor& x = tensor("x", args[0]);
  const auto dt = x.scalar_type();
  if (dt != at::kBFloat16 && dt != at::kHalf) type_error("x must be bfloat16 or float16, got ", dt);
  if (!x.is_cuda()) value_error("x must be a device tensor (the 4-bit path has no CPU implementation)");
  if (x.dim() != 2 || !unit_stride(x) || x.size(1) < 1)
    value_error("x must be [M, K] with contiguous rows, got ", dims(x.sizes()), " / ", dims(x.strides()));
  Tensor w4 = tensor("w4", args[1]), scale = tensor("scale", args[2]), zero = tensor("zero", args[3], true);
  const Tensor& bias = tensor("bias", args[4], true);
  const std::string fmt = word("fmt", args[6]);
  if ((fmt != "int4" && fmt != "fp4") || (zero.defined() && fmt != "int4"))
    value_error("fmt must be 'int4' or 'fp4' (zeros: 'int4' only), got '", fmt, "'");
  const int64_t m = x.size(0), k = x.size(1);
  if (w4.dim() != 3 || scale.dim() != 4) value_error("w4 and scale must be [N/16, K/128, 1024] and [N/16, K/128, 16, groups]");
  const int64_t n = args[5] == Py_None ? 16 * w4.size(0) : integer("out_features", args[5]);
  const int64_t nt = (n + 15) / 16, kt = (k + 127) / 128, per = scale.size(3);
  if (n < 1 || w4.scalar_type() != at::kByte || w4.sizes() != at::IntArrayRef({nt, kt, 1024}) || !w4.is_contiguous())
    value_error("w4 must be contiguous uint8 ", dims({nt, kt, 1024}), " for ", n, " x ", k, ", got ", w4.scalar_type(), " ", dims(w4.sizes()));
  if (per != 1 && per != 2 && per != 4) value_error("groups must be of 32, 64 or 128 columns, got scales ", dims(scale.sizes()));
  const std::array<int64_t, 4> groups = {nt, kt, 16, per};
  if (scale.scalar_type() != at::kBFloat16 || scale.sizes() != at::IntArrayRef(groups) || !scale.is_contiguous())
    value_error("scale must be contiguous bfloat16 ", dims(groups), ", got ", scale.scalar_type(), " ", dims(scale.sizes()));
  if (zero.defined() && (zero.scalar_type() != at::kByte || zero.sizes() != at::IntArrayRef(groups) || !zero.is_contiguous()))
    value_error("zero must be contiguous uint8 ", dims(groups), ", got ", zero.scalar_type(), " ", dims(zero.sizes()));
  if (bias.defined() && (bias.scalar_type() != dt || bias.dim() != 1 || bias.size(0) != n || !bias.is_contiguous()))
    value_error("bias must be contiguous ", dt, " (", n, ",), got ", bias.scalar_type(), " ", dims(bias.sizes()));
  same_device("gemm_w4", x, w4, scale, zero, bias);
  const On on(x);
  // weights at an address the kernel does not load from (views of a larger buffer) as copies
  for (Tensor* t : {&w4, &scale, &zero})
    if (t->defined() && (uintptr_t)t->data_ptr() % 16) *t = t->clone();
  Tensor out = at::empty({m, n}, x.options());
  if (m)
    done(lbw_gemm_w4(x.data_ptr(), dt == at::kHalf ? LBW_DTYPE_FP16 : LBW_DTYPE_BF16, m, k, x.stride(0), (const uint8_t*)w4.data_ptr(),
                     (const uint16_t*)scale.data_ptr(), (const uint8_t*)ptr(zero), fmt == "fp4" ? LBW_W4_FP4 : LBW_W4_INT4,
                     128 / per, n, ptr(bias), out.data_ptr(), on.stream),
         "lbw_gemm_w4");
  return wrap(out);
  END_HANDLE_TH_ERRORS
}

// Whether a kernel may take these tensors (None: absent) by their address: none records a gradient, carries a forward-mode
// tangent, stands for others inside a torch.func transform, or is of a subclass.
PyObject* plain(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const bool grad = c10::GradMode::is_enabled();
  for (Py_ssize_t i = 0; i < n; ++i) {
    if (args[i] == Py_None) continue;
    if (!THPVariable_Check(args[i])) continue;   // (the call itself says what it wanted)
    if (!THPVariable_CheckExact(args[i])) Py_RETURN_FALSE;
    const Tensor& t = THPVariable_Unpack(args[i]);
    const auto keys = t.key_set();
    if ((grad && t.requires_grad()) || keys.has(c10::DispatchKey::FuncTorchBatched) ||
        keys.has(c10::DispatchKey::FuncTorchGradWrapper) || keys.has(c10::DispatchKey::Functionalize) || t._fw_grad(0).defined())
      Py_RETURN_FALSE;
  }
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// Whether these tensors (None: absent) are of different types.
PyObject* mixed(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Tensor* first = nullptr;
  for (Py_ssize_t i = 0; i < n; ++i) {
    if (!THPVariable_Check(args[i])) continue;
    const Tensor& t = THPVariable_Unpack(args[i]);
    if (first && first->scalar_type() != t.scalar_type()) Py_RETURN_TRUE;
    first = &t;
  }
  Py_RETURN_FALSE;
  END_HANDLE_TH_ERRORS
}

PyObject* on_status(PyObject*, PyObject* f) {
  Py_INCREF(f);
  Py_XSETREF(status_handler, f);
  Py_RETURN_NONE;
}

#define FAST(f) {#f, (PyCFunction)(void*)f, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(gated_norm), FAST(gated_norm_bwd), FAST(rotary), FAST(gemm_w4), FAST(plain), FAST(mixed),
                         {"on_status", on_status, METH_O, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_block", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__block() { return PyModule_Create(&module); }
