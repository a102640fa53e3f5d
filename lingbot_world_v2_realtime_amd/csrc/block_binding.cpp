// The block operators' calls from Python: tensors checked, outputs allocated and the C-ABI of include/lbw_block.h
// called in one native step. A call of these is bound by its host side (a token's norm takes 4 us on the GPU); the
// same checks and the 33 arguments of a ctypes call took 15-19 us in Python, against 5 here.
#include "binding.h"

namespace {

using namespace lbw_py;

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

// The options of a norm: what its gradient needs besides the tensors.
struct NormOptions : torch::CustomClassHolder {
  int norm, post, dtype, vec_dtype, rowwise = 0;
  float eps, a, b;
  int64_t batch, len, width, groups = 1, group_len;
};

struct Norm {
  static constexpr int ARGS = 2 + VECTORS + 6;
  Tensor x, y, v[VECTORS];
  c10::intrusive_ptr<NormOptions> o;

  Norm() = default;
  // x, y, the vectors, norm, post_norm, eps, residual_scale, branch_scale, group_len, checked
  explicit Norm(PyObject* const* args) : x(tensor("x", args[0])), y(tensor("y", args[1], true)), o(c10::make_intrusive<NormOptions>()) {
    for (int i = 0; i < VECTORS; ++i) v[i] = tensor(VECTOR_NAMES[i], args[2 + i], true);
    args += 2 + VECTORS;
    o->dtype = o->vec_dtype = row_format("x", x);
    if (x.dim() != 3 || !unit_stride(x) || x.size(2) < 1 || x.size(2) > LBW_NORM_MAX_WIDTH)
      value_error("x must be [B, L, C] with contiguous channels, C up to ", LBW_NORM_MAX_WIDTH, ", got ", dims(x.sizes()), " / ",
                  dims(x.strides()));
    o->batch = x.size(0), o->len = x.size(1), o->width = x.size(2);
    o->norm = norm_kind("norm", args[0]), o->post = norm_kind("post_norm", args[1]);
    o->eps = (float)number("eps", args[2]), o->a = (float)number("residual_scale", args[3]);
    o->b = (float)number("branch_scale", args[4]);
    if (y.defined()) {
      if (y.scalar_type() != x.scalar_type()) type_error("x (", x.scalar_type(), ") and y (", y.scalar_type(), ") must have one dtype");
      if (y.sizes() != x.sizes() || !unit_stride(y))
        value_error("y ", dims(y.sizes()), " / ", dims(y.strides()), " must be ", dims(x.sizes()), " with contiguous channels");
    } else if (o->post || v[GATE].defined() || v[POST_WEIGHT].defined()) {
      value_error("gate, post_norm and post_weight act on the branch: give y");
    }
    if (!o->norm) {
      for (int i : {WEIGHT, BIAS, SHIFT, SCALE})
        if (v[i].defined()) value_error("weight, bias, shift and scale follow the norm: give one");
      if (!y.defined()) value_error("nothing to do: give y or a norm");
    }
    same_device("gated_norm", x, y, v[0], v[1], v[2], v[3], v[4], v[5]);
    const Tensor* first = nullptr;
    int64_t rows = -1;
    for (int i = 0; i < VECTORS; ++i) {
      const Tensor& t = v[i];
      if (!t.defined()) continue;
      const auto d = t.scalar_type();
      if ((d != x.scalar_type() && d != at::kFloat) || (first && d != first->scalar_type()))
        type_error("the vectors must all be ", x.scalar_type(), " or all float32, got ", VECTOR_NAMES[i], " of ", d);
      first = &t;
      const bool many = i <= SCALE && t.dim() == 3;
      if (!unit_stride(t) || !(many ? t.size(0) == o->batch && t.size(2) == o->width : t.dim() == 1 && t.size(0) == o->width))
        value_error(VECTOR_NAMES[i], " must be [", o->width, "]",
                    i <= SCALE ? text(" or [", o->batch, ", rows, ", o->width, "]") : "", " with contiguous channels, got ",
                    dims(t.sizes()), " / ", dims(t.strides()));
      if (!many) continue;
      o->rowwise |= 1 << i;
      if (rows >= 0 && rows != t.size(1)) value_error("modulation vectors with ", rows, " and ", t.size(1), " rows");
      rows = t.size(1);
    }
    if (first) o->vec_dtype = row_format("vectors", *first);
    const int64_t len = o->len;
    if (rows < 0) {
      if (args[5] != Py_None) value_error("group_len is for modulation vectors with rows ([B, rows, C])");
      o->group_len = len > 0 ? len : 1;
      return;
    }
    if (rows < 1) value_error("modulation vectors need a row at least");
    o->groups = rows;
    o->group_len = args[5] == Py_None ? std::max<int64_t>((len + rows - 1) / rows, 1) : integer("group_len", args[5]);
    if (o->group_len < 1 || o->group_len > (1 << 30) || (len + o->group_len - 1) / o->group_len > rows)
      value_error(rows, " modulation rows of ", o->group_len, " tokens do not cover ", len, " tokens");
  }
  int64_t stride(int i, int dim) const { return o->rowwise >> i & 1 ? v[i].stride(dim) : 0; }
  bool empty() const { return o->batch * o->len == 0; }
  int64_t y_stride(int dim) const { return y.defined() ? y.stride(dim) : 0; }

  // (s or none, h or none)
  std::array<Tensor, 2> forward(bool want_stream) const {
    Tensor s = want_stream || !o->norm ? new_like(x) : Tensor(), h = o->norm ? new_like(x) : Tensor();
    if (!empty()) {
      const On on(x);
      done(lbw_gated_norm(x.data_ptr(), ptr(y), o->dtype, o->vec_dtype, o->batch, o->len, o->width, x.stride(0), x.stride(1),
                          y_stride(0), y_stride(1), ptr(v[GATE]), stride(GATE, 0), stride(GATE, 1), ptr(v[SHIFT]),
                          stride(SHIFT, 0), stride(SHIFT, 1), ptr(v[SCALE]), stride(SCALE, 0), stride(SCALE, 1), o->group_len,
                          ptr(v[WEIGHT]), ptr(v[BIAS]), ptr(v[POST_WEIGHT]), o->norm, o->post, o->eps, o->a, o->b, ptr(s),
                          ptr(h), on.stream),
           "lbw_gated_norm");
    }
    return {s, h};
  }

  // The gradients of x, y and the vectors, those with their bit in `wants`. ds and dh are packed, of x's type and
  // shape.
  std::array<Tensor, 2 + VECTORS> backward(const Tensor& ds, const Tensor& dh, int64_t wants, bool python) const {
    std::array<Tensor, 2 + VECTORS> g;
    void* p[2 + VECTORS] = {};
    bool sums = false;
    const bool none = (!ds.defined() && !dh.defined()) || empty();
    for (int i = 0; i < 2 + VECTORS; ++i) {
      const Tensor& t = i == 0 ? x : i == 1 ? y : v[i - 2];
      if (!(wants >> i & 1) || !t.defined()) continue;
      // what only the norm's output depends on has a gradient of zero without dh
      const bool idle = none || (!dh.defined() && i >= 2 + SHIFT && i <= 2 + BIAS);
      g[i] = idle ? at::zeros(t.sizes(), t.options()) : new_like(t);
      if (idle) continue;
      p[i] = g[i].data_ptr();
      sums = sums || i >= 2;
    }
    if (none) return g;
    const On on(x);
    Tensor ws;
    if (sums)
      ws = at::empty({lbw_gated_norm_bwd_workspace_bytes(o->batch, o->len, o->width, o->groups, o->group_len)},
                     x.options().dtype(at::kByte));
    done(lbw_gated_norm_bwd(ptr(ds), ptr(dh), x.data_ptr(), ptr(y), o->dtype, o->vec_dtype, o->batch, o->len, o->width,
                            x.stride(0), x.stride(1), y_stride(0), y_stride(1), ptr(v[GATE]), stride(GATE, 0), stride(GATE, 1),
                            ptr(v[SCALE]), stride(SCALE, 0), stride(SCALE, 1), o->rowwise, o->groups, o->group_len,
                            ptr(v[WEIGHT]), ptr(v[BIAS]), ptr(v[POST_WEIGHT]), o->norm, o->post, o->eps, o->a, o->b, p[0], p[1],
                            p[2 + GATE], p[2 + SHIFT], p[2 + SCALE], p[2 + WEIGHT], p[2 + BIAS], p[2 + POST_WEIGHT], ptr(ws),
                            on.stream),
         "lbw_gated_norm_bwd", python);
    return g;
  }
};

struct NormFunction : torch::autograd::Function<NormFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Maybe& y, const Maybe&, const Maybe&, const Maybe&,
                               const Maybe&, const Maybe&, const Maybe&, const Norm* a) {
    ctx->set_materialize_grads(false);
    variable_list kept = {a->x, a->y};
    kept.insert(kept.end(), a->v, a->v + VECTORS);
    ctx->save_for_backward(kept);
    ctx->saved_data["options"] = c10::IValue::make_capsule(a->o);
    variable_list out;
    for (const Tensor& t : a->forward(a->y.defined()))
      if (t.defined()) out.push_back(t);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    TORCH_CHECK(!c10::GradMode::is_enabled(), "gated_norm has no second derivative");
    const variable_list kept = ctx->get_saved_variables();
    Norm a;
    a.x = kept[0], a.y = kept[1];
    for (int i = 0; i < VECTORS; ++i) a.v[i] = kept[2 + i];
    a.o = c10::static_intrusive_pointer_cast<NormOptions>(ctx->saved_data["options"].toCapsule());
    int64_t wants = 0, edge = 0;
    for (int i = 0; i < 2 + VECTORS; ++i)
      if (kept[i].defined() && ctx->needs_input_grad(edge++)) wants |= 1 << i;
    for (Tensor& d : grads)
      if (d.defined()) d = d.resolve_neg().contiguous();
    const bool both = grads.size() == 2;
    const Tensor ds = both || !a.o->norm ? grads[0] : Tensor(), dh = both ? grads[1] : a.o->norm ? grads[0] : Tensor();
    const auto g = a.backward(ds, dh, wants, false);
    variable_list out(g.begin(), g.end());
    out.emplace_back();   // the call itself
    return out;
  }
};

// The operator as users call it: (s or None, h or None), with a gradient where one is recorded. Vectors of different
// types are taken in fp32.
PyObject* norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, Norm::ARGS);
  std::array<PyObject*, Norm::ARGS> own;
  std::array<THPObjectPtr, VECTORS> held;
  std::copy(args, args + Norm::ARGS, own.begin());
  const auto type = tensor("x", args[0]).scalar_type();
  bool half = false, full = false;
  for (int i = 2; i < 2 + VECTORS; ++i) {
    if (!THPVariable_Check(args[i])) continue;
    const auto d = THPVariable_Unpack(args[i]).scalar_type();
    half = half || d == type;
    full = full || d == at::kFloat;
  }
  for (int i = 2; half && full && i < 2 + VECTORS; ++i) {   // (other types stay, and are refused below)
    if (!THPVariable_Check(args[i]) || THPVariable_Unpack(args[i]).scalar_type() != type) continue;
    held[i - 2] = THPVariable_Wrap(THPVariable_Unpack(args[i]).to(at::kFloat));
    own[i] = held[i - 2].get();
  }
  const Norm a(own.data());
  if (!records_gradient(a.x, a.y, a.v[0], a.v[1], a.v[2], a.v[3], a.v[4], a.v[5]))
    return wrap_all(a.forward(a.y.defined()));
  const auto out = NormFunction::apply(a.x, maybe(a.y), maybe(a.v[0]), maybe(a.v[1]), maybe(a.v[2]), maybe(a.v[3]),
                                       maybe(a.v[4]), maybe(a.v[5]), &a);
  return wrap_all(std::array<Tensor, 2>{a.y.defined() ? out.front() : Tensor(), a.o->norm ? out.back() : Tensor()});
  END_HANDLE_TH_ERRORS
}

// The forward alone: the norm's arguments, and whether the stream is wanted.
PyObject* gated_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, Norm::ARGS + 1);
  no_gradient("kernels.gated_norm", args, n);
  return wrap_all(Norm(args).forward(truth(args[Norm::ARGS])));
  END_HANDLE_TH_ERRORS
}

// The gradients alone: the norm's arguments, ds, dh, and a bit for each of x, y and the vectors. A tuple of those,
// None for the others.
PyObject* gated_norm_bwd(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, Norm::ARGS + 3);
  no_gradient("kernels.gated_norm_bwd", args, n);
  const Norm a(args);
  const Tensor &ds = tensor("ds", args[Norm::ARGS], true), &dh = tensor("dh", args[Norm::ARGS + 1], true);
  const int64_t wants = integer("wants", args[Norm::ARGS + 2]);
  for (const auto& [name, d] : {std::pair<const char*, const Tensor&>{"ds", ds}, {"dh", dh}})
    if (d.defined() && (d.scalar_type() != a.x.scalar_type() || d.sizes() != a.x.sizes() || !d.is_contiguous()))
      value_error(name, " must be contiguous ", a.x.scalar_type(), " ", dims(a.x.sizes()), ", got ", d.scalar_type(), " ",
                  dims(d.sizes()));
  if (dh.defined() && !a.o->norm) value_error("dh without a norm");
  same_device("gated_norm_bwd", a.x, ds, dh);
  return wrap_all(a.backward(ds, dh, wants, true));
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------- rotary

// Memory that tensors share, found exactly for strided views too (torch's own check answers for packed ones only). Two
// elements share a byte where sum x_k step_k = target has a solution with lo_k <= x_k <= hi_k: a term for every
// dimension of either, and one of single bytes for the elements' size.
class Overlap {
  struct Term {
    int64_t step, lo, hi;
  };
  static constexpr int MOST = 2 * 4 + 1;      // (4-d tensors)
  Term terms[MOST];                           // steps falling, the bytes last
  int64_t low[MOST + 1], high[MOST + 1];      // least and largest sum of the terms from k on
  int n = 0, budget = 1 << 16;                // looks, after which the answer is that they might

  void add(const Tensor& t, bool first, bool second) {
    const int64_t size = t.element_size();
    for (int i = 0; i < 4; ++i) {
      const int64_t most = t.size(i) - 1;
      if (most > 0) terms[n++] = {t.stride(i) * size, second ? -most : 0, first ? most : 0};
    }
  }
  // dimensions of one step as one: views of one projection share theirs, and each place of the one would be tried
  // with the nearest of the other (a chunk's tokens would spend the budget)
  void merge() {
    int m = 0;
    for (int i = 0; i < n; ++i) {
      int j = 0;
      while (j < m && terms[j].step != terms[i].step) ++j;
      if (j < m) {
        terms[j].lo += terms[i].lo;
        terms[j].hi += terms[i].hi;
      } else {
        terms[m++] = terms[i];
      }
    }
    n = m;
  }
  void sort(int64_t size) {
    std::sort(terms, terms + n, [](const Term& a, const Term& b) { return a.step > b.step; });
    terms[n++] = {1, 1 - size, size - 1};
    low[n] = high[n] = 0;
    for (int k = n; k-- > 0;) {
      low[k] = low[k + 1] + terms[k].lo * terms[k].step;
      high[k] = high[k + 1] + terms[k].hi * terms[k].step;
    }
  }
  static int64_t floor_div(int64_t a, int64_t b) { return a / b - (a % b < 0); }
  // whether the terms from k on reach `target`
  bool reach(int k, int64_t target) {
    if (target < low[k] || target > high[k]) return false;
    // (nothing but bytes, and steps of zero, left: they reach all of their range)
    if (k + 1 == n || terms[k].step == 0 || --budget < 0) return true;
    const Term& t = terms[k];
    const int64_t x0 = std::max(t.lo, -floor_div(high[k + 1] - target, t.step)), x1 = std::min(t.hi, floor_div(target - low[k + 1], t.step));
    for (int64_t x = x0; x <= x1; ++x)
      if (reach(k + 1, target - x * t.step)) return true;
    return false;
  }

 public:
  static bool of(const Tensor& a, const Tensor& b) {
    if (!a.defined() || !b.defined() || !a.numel() || !b.numel() || a.device() != b.device()) return false;
    Overlap o;
    o.add(a, true, false);
    o.add(b, false, true);
    o.merge();
    o.sort(a.element_size());
    return o.reach(0, (const char*)b.data_ptr() - (const char*)a.data_ptr());
  }
  // whether two elements of `t` share memory: two places that differ, by more in the k-th term than by nothing
  static bool within(const Tensor& t) {
    if (!t.defined() || !t.numel()) return false;
    Overlap o;
    o.add(t, true, true);
    o.sort(t.element_size());
    for (int k = 0; k + 1 < o.n; ++k) {
      const Term& d = o.terms[k];
      if (d.step == 0) return true;
      for (int64_t x = 1; x <= d.hi && x * d.step <= o.high[k + 1]; ++x)
        if (o.reach(k + 1, -x * d.step)) return true;
    }
    return false;
  }
};

// Tensors of which one is written while the other is read or written, by different threads.
void apart(const Tensor& a, const Tensor& b, const char* what) {
  if (Overlap::of(a, b)) value_error(what, " share their memory");
}

// An output: every element has memory of its own.
void own_memory(const Tensor& t, const char* name) {
  if (Overlap::within(t)) value_error(name, " has elements that share their memory");
}

bool same_memory(const Tensor& a, const Tensor& b) {   // (of one shape)
  bool same = a.data_ptr() == b.data_ptr();
  for (int64_t i = 0; i < a.dim(); ++i) same = same && (a.size(i) <= 1 || a.stride(i) == b.stride(i));
  return same;
}

// A tensor written in place: a graph that kept it notices.
void written(const Tensor& t) {
  if (t.defined() && !t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

struct RotaryFunction : torch::autograd::Function<RotaryFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Maybe& k, const Rotary* a) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({a->pos, a->freq, a->axis});
    ctx->saved_data["options"] = c10::IValue::make_capsule(a->o);
    ctx->saved_data["k"] = a->k.defined();
    const auto out = a->fresh(false, true);
    return a->k.defined() ? variable_list{out[0], out[1]} : variable_list{out[0]};
  }
  // the opposite rotation of whichever gradients there are (one rotation takes any number of heads)
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    TORCH_CHECK(!c10::GradMode::is_enabled(), "rotary_embed has no second derivative");
    const variable_list kept = ctx->get_saved_variables();
    Rotary a;
    a.pos = kept[0], a.freq = kept[1], a.axis = kept[2];
    a.o = c10::static_intrusive_pointer_cast<RotaryOptions>(ctx->saved_data["options"].toCapsule());
    Tensor d[2];
    for (size_t i = 0; i < grads.size(); ++i)
      if (grads[i].defined() && ctx->needs_input_grad(i)) {
        d[i] = grads[i].resolve_neg();
        if (!unit_stride(d[i])) d[i] = d[i].contiguous();
      }
    variable_list out(3);
    if (!d[0].defined() && !d[1].defined()) return out;
    const bool q = d[0].defined();
    a.q = q ? d[0] : d[1];
    if (q) a.k = d[1];
    const auto g = a.fresh(true, false);
    if (q) out[0] = g[0];
    out[1] = q ? g[1] : g[0];
    return out;
  }
};

// The operator as users call it: q, k, positions, freq, axis, pairs, factor, layout, axes, inplace. (q, k or None), with
// a gradient where one is recorded.
PyObject* rotary_embed(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 10);
  const Rotary a(args);
  const bool grad = records_gradient(a.q, a.k);
  if (truth(args[9])) {
    if (grad) value_error("q and k cannot be rotated in place where a gradient is recorded");
    own_memory(a.q, "q");
    own_memory(a.k, "k");
    apart(a.q, a.k, "q and k, to be rotated in place,");
    a.run(a.q, a.k, false, true);
    written(a.q);
    written(a.k);
    return wrap_all(std::array<Tensor, 2>{a.q, a.k});
  }
  if (!grad) return wrap_all(a.fresh(false, true));
  const auto out = RotaryFunction::apply(a.q, maybe(a.k), &a);
  return wrap_all(std::array<Tensor, 2>{out[0], a.k.defined() ? out[1] : Tensor()});
  END_HANDLE_TH_ERRORS
}

// The rotation alone: q, k, positions, freq, axis, pairs, factor, layout, axes, inverse, q_out, k_out.
PyObject* rotary(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 12);
  no_gradient("kernels.rotary", args, n);
  const Rotary a(args);
  std::array<Tensor, 2> out;
  for (int i = 0; i < 2; ++i) {
    const Tensor &x = i ? a.k : a.q, &o = tensor(i ? "k_out" : "q_out", args[10 + i], true);
    const char* name = i ? "k_out" : "q_out";
    if (!x.defined()) {
      if (o.defined()) value_error("k_out without k");
      continue;
    }
    out[i] = o.defined() ? o : new_like(x);
    if (!o.defined()) continue;
    if (o.scalar_type() != x.scalar_type() || o.sizes() != x.sizes() || !unit_stride(o))
      value_error(name, " must be ", x.scalar_type(), " ", dims(x.sizes()), " with contiguous channels");
    own_memory(o, name);
    if (!same_memory(o, x) && Overlap::of(o, x)) value_error(name, " overlaps its input, but is not the input itself");
  }
  same_device("rotary", a.q, out[0], out[1]);
  apart(out[0], out[1], "q_out and k_out");
  apart(out[0], a.k, "q_out and k");
  apart(out[1], a.q, "k_out and q");
  a.run(out[0], out[1], truth(args[9]), true);
  written(out[0]);
  written(out[1]);
  return wrap_all(out);
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------- 4-bit linears

// x, w4, scale, zero, bias, out_features, fmt, whether the bias may be fp32 (else it has x's type)
PyObject* gemm_w4(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  count(n_args, 8);
  const Tensor& x = tensor("x", args[0]);
  const auto dt = x.scalar_type();
  if (dt != at::kBFloat16 && dt != at::kHalf) type_error("x must be bfloat16 or float16, got ", dt);
  if (x.dim() != 2 || !unit_stride(x) || x.size(1) < 1)
    value_error("x must be [M, K] with contiguous rows, got ", dims(x.sizes()), " / ", dims(x.strides()));
  Tensor w4 = tensor("w4", args[1]), scale = tensor("scale", args[2]), zero = tensor("zero", args[3], true);
  const Tensor& bias = tensor("bias", args[4], true);
  no_gradient("gemm_w4", records_gradient(x, scale, bias));
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
  const bool bias_fp32 = bias.defined() && bias.scalar_type() == at::kFloat && truth(args[7]);
  if (bias.defined() && ((bias.scalar_type() != dt && !bias_fp32) || bias.dim() != 1 || bias.size(0) != n || !bias.is_contiguous()))
    value_error("bias must be contiguous ", dt, " (", n, ",), got ", bias.scalar_type(), " ", dims(bias.sizes()));
  if (!x.is_cuda()) value_error("x must be a device tensor (the 4-bit path has no CPU implementation)");
  same_device("gemm_w4", x, w4, scale, zero, bias);
  const On on(x);
  // weights at an address the kernel does not load from (views of a larger buffer) as copies
  for (Tensor* t : {&w4, &scale, &zero})
    if (t->defined() && (uintptr_t)t->data_ptr() % 16) *t = t->clone();
  Tensor out = at::empty({m, n}, x.options());
  if (m)
    done(lbw_gemm_w4(x.data_ptr(), (dt == at::kHalf ? LBW_DTYPE_FP16 : LBW_DTYPE_BF16) + (bias_fp32 ? LBW_W4_BIAS_FP32 : 0), m, k, x.stride(0), (const uint8_t*)w4.data_ptr(),
                     (const uint16_t*)scale.data_ptr(), (const uint8_t*)ptr(zero), fmt == "fp4" ? LBW_W4_FP4 : LBW_W4_INT4,
                     128 / per, n, ptr(bias), out.data_ptr(), on.stream),
         "lbw_gemm_w4");
  return wrap(out);
  END_HANDLE_TH_ERRORS
}

bool in_transform(const Tensor& t) {
  const auto keys = t.key_set();
  return keys.has(c10::DispatchKey::FuncTorchBatched) || keys.has(c10::DispatchKey::FuncTorchGradWrapper) ||
         keys.has(c10::DispatchKey::Functionalize);
}

// The input of a 4-bit linear, refused where the kernel may not take it by its address or would lose its gradient.
PyObject* linear_input(PyObject*, PyObject* x) {
  HANDLE_TH_ERRORS
  if (!THPVariable_Check(x)) type_error("W4Linear takes a tensor, got ", Py_TYPE(x)->tp_name);
  if (!THPVariable_CheckExact(x)) type_error("W4Linear takes no tensor subclass, got ", Py_TYPE(x)->tp_name);
  const Tensor& t = THPVariable_Unpack(x);
  const char* why = in_transform(t) ? "W4Linear does not run inside a torch.func transform"
      : c10::GradMode::is_enabled() && t.requires_grad()
          ? "W4Linear has no gradient with respect to its input: call it under torch.no_grad(), or on a detached input"
      : records_gradient(t) ? "W4Linear has no derivative for a forward-mode tangent: call it on a detached input"
                            : nullptr;
  if (why) {
    PyErr_SetString(PyExc_RuntimeError, why);
    throw python_error();
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// Whether a kernel may take these tensors (None: absent) by their address: none records a gradient, carries a
// forward-mode tangent, stands for others inside a torch.func transform, or is of a subclass.
PyObject* plain(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  for (Py_ssize_t i = 0; i < n; ++i) {
    if (args[i] == Py_None) continue;
    if (!THPVariable_Check(args[i])) continue;   // (the call itself says what it wanted)
    if (!THPVariable_CheckExact(args[i])) Py_RETURN_FALSE;
    const Tensor& t = THPVariable_Unpack(args[i]);
    if (in_transform(t) || records_gradient(t)) Py_RETURN_FALSE;
  }
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

PyObject* on_status(PyObject*, PyObject* f) {
  Py_INCREF(f);
  Py_XSETREF(status_handler, f);
  Py_RETURN_NONE;
}

#define FAST(f) {#f, (PyCFunction)(void*)f, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(norm), FAST(gated_norm), FAST(gated_norm_bwd), FAST(rotary_embed), FAST(rotary), FAST(gemm_w4),
                         FAST(plain), FAST(norm_rotary_embed), FAST(packed_attention), FAST(kv4_write), FAST(kv4_read),
                         FAST(kv4_attend),
                         {"linear_input", linear_input, METH_O, nullptr},
                         {"on_status", on_status, METH_O, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_block", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__block() { return PyModule_Create(&module); }
