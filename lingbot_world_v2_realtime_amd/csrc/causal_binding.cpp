// The calls of causal self-attention from Python (include/lbw_causal.h): norms with rotation, packed attention, and the
// cache in 4 bits. Part of _block.so; block_binding.cpp says why these are native.
#include "binding.h"

namespace lbw_py {

namespace {

// ---------------------------------------------------------------- norm and rotation by head

// The rotation's arguments with the weights: lbw_norm_rotary and its gradient.
struct NormRotary : Rotary {
  Tensor weight[2];
  int vec_dtype = 0;
  float eps = 0;

  NormRotary() = default;
  // q, k, positions, freq, axis, pairs, factor, layout, axes, q_weight, k_weight, eps
  explicit NormRotary(PyObject* const* args) : Rotary(args) {
    vec_dtype = element_format("q", q);
    for (int i = 0; i < 2; ++i) {
      const char* name = i ? "k_weight" : "q_weight";
      const Tensor& t = weight[i] = tensor(name, args[9 + i], true);
      if (!t.defined()) continue;
      if (i && !k.defined()) value_error("k_weight without k");
      if (t.scalar_type() != q.scalar_type() && t.scalar_type() != at::kFloat)
        type_error(name, " must be ", q.scalar_type(), " or float32, got ", t.scalar_type());
      if (i && weight[0].defined() && weight[0].scalar_type() != t.scalar_type())
        type_error("q_weight (", weight[0].scalar_type(), ") and k_weight (", t.scalar_type(), ") must have one dtype");
      if (t.dim() != 1 || t.size(0) != q.size(3) || !t.is_contiguous())
        value_error(name, " must be contiguous (", q.size(3), ",), got ", dims(t.sizes()), " / ", dims(t.strides()));
      vec_dtype = element_format(name, t);
    }
    eps = (float)number("eps", args[11]);
    if (!(eps >= 0.f)) value_error("eps must not be negative, got ", eps);
    same_device("norm_rotary_embed", q, k, weight[0], weight[1]);
  }
  int64_t st(const Tensor& t, int dim) const { return t.defined() ? t.stride(dim) : 0; }
  bool empty() const { return q.numel() + (k.defined() ? k.numel() : 0) == 0; }
  int64_t own() const { return pos.defined() ? own_dims() : 0; }

  std::array<Tensor, 2> forward() const {
    on_device("q", q);
    const std::array<Tensor, 2> out = {new_like(q), k.defined() ? new_like(k) : Tensor()};
    if (empty()) return out;
    const On on(q);
    const auto w = weights();
    done(lbw_norm_rotary(q.data_ptr(), ptr(k), element_format("q", q), vec_dtype, q.size(0), q.size(tok()), q.size(head()),
                         k.defined() ? k.size(head()) : 0, q.size(3), freq.size(0), st(q, 0), st(q, tok()), st(q, head()), st(k, 0),
                         st(k, tok()), st(k, head()), ptr(w[0]), ptr(w[1]), eps, ptr(pos),
                         pos.defined() && pos.scalar_type() == at::kLong, own() == 2 ? pos.stride(0) : 0, own() ? pos.stride(own() - 1) : 0,
                         own() && axis.defined() ? pos.stride(own()) : 0, o->start, (const double*)freq.data_ptr(),
                         (const int32_t*)ptr(axis), own() && axis.defined() ? pos.size(own()) : 1, o->interleaved, (float)o->factor,
                         out[0].data_ptr(), ptr(out[1]), st(out[0], 0), st(out[0], tok()), st(out[0], head()), st(out[1], 0),
                         st(out[1], tok()), st(out[1], head()), on.stream),
         "lbw_norm_rotary");
    return out;
  }
  // weights at an address that the kernels do not load from (views of a larger buffer) as copies
  std::array<Tensor, 2> weights() const {
    std::array<Tensor, 2> w = {weight[0], weight[1]};
    for (Tensor& t : w)
      if (t.defined() && (uintptr_t)t.const_data_ptr() % 16) t = t.clone();
    return w;
  }
  // The gradients of q, k and the weights, those that are wanted, from the outputs' (either may be undefined).
  std::array<Tensor, 4> backward(const Tensor& dq, const Tensor& dk, const std::array<bool, 4>& wants) const {
    std::array<Tensor, 4> g;
    const bool none = empty() || (!dq.defined() && !dk.defined());
    const Tensor* of[4] = {&q, &k, &weight[0], &weight[1]};
    for (int i = 0; i < 4; ++i)
      if (wants[i] && of[i]->defined()) g[i] = none ? at::zeros(of[i]->sizes(), of[i]->options()) : new_like(*of[i]);
    if (none) return g;
    const On on(q);
    const auto w = weights();
    Tensor ws;
    if (g[2].defined() || g[3].defined())
      ws = at::empty({lbw_norm_rotary_bwd_workspace_bytes(q.size(3))}, q.options().dtype(at::kByte));
    const Tensor &oq = g[0].defined() ? g[0] : absent, &ok = g[1].defined() ? g[1] : absent;
    done(lbw_norm_rotary_bwd(ptr(dq), ptr(dk), q.data_ptr(), ptr(k), element_format("q", q), vec_dtype, q.size(0), q.size(tok()),
                             q.size(head()), k.defined() ? k.size(head()) : 0, q.size(3), freq.size(0), st(dq, 0), st(dq, tok()),
                             st(dq, head()), st(dk, 0), st(dk, tok()), st(dk, head()), st(q, 0), st(q, tok()), st(q, head()), st(k, 0),
                             st(k, tok()), st(k, head()), ptr(w[0]), ptr(w[1]), eps, ptr(pos),
                             pos.defined() && pos.scalar_type() == at::kLong, own() == 2 ? pos.stride(0) : 0,
                             own() ? pos.stride(own() - 1) : 0, own() && axis.defined() ? pos.stride(own()) : 0, o->start,
                             (const double*)freq.data_ptr(), (const int32_t*)ptr(axis), own() && axis.defined() ? pos.size(own()) : 1,
                             o->interleaved, (float)o->factor, ptr(oq), ptr(ok), st(oq, 0), st(oq, tok()), st(oq, head()), st(ok, 0),
                             st(ok, tok()), st(ok, head()), ptr(g[2]), ptr(g[3]), ptr(ws), on.stream),
         "lbw_norm_rotary_bwd", false);
    return g;
  }
};

struct NormRotaryFunction : torch::autograd::Function<NormRotaryFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Maybe& k, const Maybe& q_weight, const Maybe& k_weight,
                               const NormRotary* a) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({a->q, a->k, a->weight[0], a->weight[1], a->pos, a->freq, a->axis});
    ctx->saved_data["options"] = c10::IValue::make_capsule(a->o);
    ctx->saved_data["vec"] = (int64_t)a->vec_dtype;
    ctx->saved_data["eps"] = (double)a->eps;
    const auto out = a->forward();
    return a->k.defined() ? variable_list{out[0], out[1]} : variable_list{out[0]};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    TORCH_CHECK(!c10::GradMode::is_enabled(), "norm_rotary_embed has no second derivative");
    const variable_list kept = ctx->get_saved_variables();
    NormRotary a;
    a.q = kept[0], a.k = kept[1], a.weight[0] = kept[2], a.weight[1] = kept[3], a.pos = kept[4], a.freq = kept[5], a.axis = kept[6];
    a.o = c10::static_intrusive_pointer_cast<RotaryOptions>(ctx->saved_data["options"].toCapsule());
    a.vec_dtype = (int)ctx->saved_data["vec"].toInt();
    a.eps = (float)ctx->saved_data["eps"].toDouble();
    // (the inputs that are tensors are counted, those absent are not)
    std::array<bool, 4> wants = {};
    int edge = 0;
    for (int i = 0; i < 4; ++i)
      if (kept[i].defined()) wants[i] = ctx->needs_input_grad(edge++);
    Tensor d[2];
    for (size_t i = 0; i < grads.size(); ++i)
      if (grads[i].defined()) {
        d[i] = grads[i].resolve_neg();
        if (!unit_stride(d[i])) d[i] = d[i].contiguous();
      }
    variable_list out(5);
    const auto g = a.backward(d[0], d[1], wants);
    std::copy(g.begin(), g.end(), out.begin());
    return out;
  }
};

// ---------------------------------------------------------------- packed sequences

// A row tensor [T, H, D] of 16-bit values that the kernels take as it is, or a copy of it: rows 16-byte aligned, channels
// next to each other, tokens apart.
bool rows_fit(const Tensor& t) {
  return unit_stride(t) && (uintptr_t)t.const_data_ptr() % 16 == 0 &&
      (t.size(0) <= 1 || (t.stride(0) % 8 == 0 && t.stride(0) >= t.size(2) && t.stride(0) < 1 << 24)) &&
      (t.size(1) <= 1 || t.stride(1) % 8 == 0);
}
Tensor rows_of(const Tensor& t) { return rows_fit(t) ? t : t.clone(at::MemoryFormat::Contiguous); }
int64_t tok_stride(const Tensor& t) { return t.size(0) <= 1 ? t.size(2) : t.stride(0); }
int64_t head_stride(const Tensor& t) { return t.size(1) <= 1 ? 0 : t.stride(1); }

int half_format(const char* name, const Tensor& t) {
  const auto d = t.scalar_type();
  if (d != at::kBFloat16 && d != at::kHalf) type_error(name, " must be bfloat16 or float16, got ", d);
  return d == at::kHalf ? LBW_DTYPE_FP16 : LBW_DTYPE_BF16;
}

const Tensor& row_tensor(const char* name, PyObject* o) {
  const Tensor& t = tensor(name, o);
  half_format(name, t);
  if (t.dim() != 3) value_error(name, " must be [rows, heads, channels], got ", dims(t.sizes()));
  if (t.size(2) != 64 && t.size(2) != 128) value_error(name, " must have heads of 64 or 128 channels, got ", dims(t.sizes()));
  if (t.size(0) >= int64_t(1) << 31) value_error(name, " has 2^31 rows or more");
  if (t.size(1) < 1 || t.size(1) > 4096) value_error(name, " must have 1 to 4096 heads, got ", t.size(1));
  return t;
}

const Tensor& starts_tensor(const char* name, PyObject* o) {
  const Tensor& t = tensor(name, o);
  if (t.scalar_type() != at::kInt) type_error(name, " must be int32, got ", t.scalar_type());
  if (t.dim() != 1 || t.size(0) < 2 || t.size(0) > 65536 || !t.is_contiguous())
    value_error(name, " must be contiguous [sequences + 1] for 1 to 65535 sequences, got ", dims(t.sizes()), " / ", dims(t.strides()));
  return t;
}

float scale_of(PyObject* o, int64_t dim) {
  if (o == Py_None) return 1.f / std::sqrt((float)dim);
  const float s = (float)number("sm_scale", o);
  if (!(s > 0.f) || !(s < std::numeric_limits<float>::infinity())) value_error("sm_scale must be positive and finite, got ", s);
  return s;
}

struct Packed {
  Tensor q, k, v, starts, k_starts;
  float scale = 0;
  bool causal = true;

  Packed() = default;
  // q, k, v, starts, k_starts, sm_scale, causal
  explicit Packed(PyObject* const* args)
      : q(row_tensor("q", args[0])), k(row_tensor("k", args[1])), v(row_tensor("v", args[2])), starts(starts_tensor("starts", args[3])) {
    k_starts = args[4] == Py_None ? starts : starts_tensor("k_starts", args[4]);
    if (k_starts.size(0) != starts.size(0)) value_error("starts ", dims(starts.sizes()), " and k_starts ", dims(k_starts.sizes()), " do not match");
    if (k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type())
      type_error("q (", q.scalar_type(), "), k (", k.scalar_type(), ") and v (", v.scalar_type(), ") must have one dtype");
    if (k.sizes() != v.sizes() || k.size(2) != q.size(2))
      value_error("q ", dims(q.sizes()), ", k ", dims(k.sizes()), ", v ", dims(v.sizes()), " do not match");
    if (q.size(1) % k.size(1)) value_error(q.size(1), " heads of q cannot share ", k.size(1), " of k and v evenly");
    if (args[4] == Py_None && q.size(0) != k.size(0))
      value_error("q ", dims(q.sizes()), " and k ", dims(k.sizes()), " have other rows: give k_starts");
    scale = scale_of(args[5], q.size(2));
    causal = truth(args[6]);
    same_device("packed_attention", q, k, v, starts, k_starts);
  }
  int64_t seqs() const { return starts.size(0) - 1; }

  // (what a gradient needs beside the output: kept = {rest, lse})
  Tensor forward(std::array<Tensor, 2>* kept) const {
    on_device("q", q);
    Tensor out = new_like(q);
    if (q.size(0) == 0) return out;
    const On on(q);
    const Tensor qr = rows_of(q), kr = rows_of(k), vr = rows_of(v);
    if (kept) *kept = {new_like(q), at::empty({q.size(1), q.size(0)}, q.options().dtype(at::kFloat))};
    done(lbw_packed_attn_fwd(qr.data_ptr(), ptr(kr), ptr(vr), half_format("q", q), seqs(), q.size(0), k.size(0), q.size(1), k.size(1),
                             q.size(2), tok_stride(qr), head_stride(qr), tok_stride(kr), head_stride(kr), tok_stride(vr),
                             head_stride(vr), (const int32_t*)starts.data_ptr(), (const int32_t*)k_starts.data_ptr(), causal, scale,
                             out.data_ptr(), kept ? (*kept)[0].data_ptr() : nullptr, kept ? (float*)(*kept)[1].data_ptr() : nullptr, on.stream),
         "lbw_packed_attn_fwd");
    return out;
  }
  std::array<Tensor, 3> backward(const Tensor& d_out, const Tensor& out, const Tensor& rest, const Tensor& lse, bool want_q, bool want_kv) const {
    std::array<Tensor, 3> g;
    const bool none = q.size(0) == 0 || k.size(0) == 0;
    if (want_q) g[0] = none ? at::zeros(q.sizes(), q.options()) : new_like(q);
    if (want_kv)
      for (int i = 1; i < 3; ++i) g[i] = none ? at::zeros(k.sizes(), k.options()) : new_like(k);
    if (none) return g;
    const On on(q);
    const Tensor qr = rows_of(q), kr = rows_of(k), vr = rows_of(v), dr = rows_of(d_out);
    const Tensor ws = at::empty({lbw_packed_attn_bwd_workspace_bytes(q.size(0), k.size(0), q.size(1), k.size(1))}, q.options().dtype(at::kByte));
    done(lbw_packed_attn_bwd(dr.data_ptr(), out.data_ptr(), rest.data_ptr(), (const float*)lse.data_ptr(), qr.data_ptr(), kr.data_ptr(), vr.data_ptr(),
                             half_format("q", q), seqs(), q.size(0), k.size(0), q.size(1), k.size(1), q.size(2), tok_stride(dr),
                             head_stride(dr), tok_stride(qr), head_stride(qr), tok_stride(kr), head_stride(kr), tok_stride(vr),
                             head_stride(vr), (const int32_t*)starts.data_ptr(), (const int32_t*)k_starts.data_ptr(), causal, scale,
                             ptr(g[0]), ptr(g[1]), ptr(g[2]), ws.data_ptr(), on.stream),
         "lbw_packed_attn_bwd", false);
    return g;
  }
};

struct PackedFunction : torch::autograd::Function<PackedFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Packed* a) {
    ctx->set_materialize_grads(false);
    std::array<Tensor, 2> more;
    const Tensor out = a->forward(&more);
    ctx->save_for_backward({a->q, a->k, a->v, a->starts, a->k_starts, out, more[0], more[1]});
    ctx->saved_data["scale"] = (double)a->scale;
    ctx->saved_data["causal"] = a->causal;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    TORCH_CHECK(!c10::GradMode::is_enabled(), "packed_attention has no second derivative");
    variable_list out(4);
    if (!grads[0].defined()) return out;
    const variable_list kept = ctx->get_saved_variables();
    Packed a;
    a.q = kept[0], a.k = kept[1], a.v = kept[2], a.starts = kept[3], a.k_starts = kept[4];
    a.scale = (float)ctx->saved_data["scale"].toDouble();
    a.causal = ctx->saved_data["causal"].toBool();
    const bool wants[3] = {ctx->needs_input_grad(0), ctx->needs_input_grad(1), ctx->needs_input_grad(2)};
    const auto g = a.backward(grads[0].resolve_neg(), kept[5], kept[6], kept[7], wants[0], wants[1] || wants[2]);
    for (int i = 0; i < 3; ++i)
      if (wants[i]) out[i] = g[i];
    return out;
  }
};

// ---------------------------------------------------------------- cache

struct Cache {
  Tensor k4, ks, v4, vs, table, lens, starts;
  int64_t layer, pages, heads, dim, rows = 0;

  // k4, ks, v4, vs, layer, table, lens, starts
  explicit Cache(PyObject* const* args)
      : k4(tensor("k", args[0])), ks(tensor("k_scale", args[1])), v4(tensor("v", args[2])), vs(tensor("v_scale", args[3])),
        table(tensor("table", args[5])), lens(tensor("lens", args[6])), starts(args[7] == Py_None ? Tensor() : starts_tensor("starts", args[7])) {
    if (k4.dim() != 5 || (k4.size(4) != 32 && k4.size(4) != 64) || k4.size(3) != LBW_KV4_PAGE || k4.size(2) < 1 || k4.size(2) > 4096 || k4.size(1) < 1)
      value_error("the cache's k must be [layers, pages, heads, 64, 32 or 64], got ", dims(k4.sizes()));
    const int64_t l = k4.size(0);
    pages = k4.size(1), heads = k4.size(2), dim = 2 * k4.size(4);
    const std::array<int64_t, 5> s5 = {l, pages, heads, LBW_KV4_PAGE, dim / 32};
    const std::array<int64_t, 4> v = {l, pages, heads, LBW_KV4_PAGE * dim / 2}, s4 = {l, pages, heads, LBW_KV4_PAGE * dim / 32};
    const struct { const char* name; const Tensor& t; at::IntArrayRef want; } parts[4] = {
        {"k", k4, k4.sizes()}, {"k_scale", ks, s5}, {"v", v4, v}, {"v_scale", vs, s4}};
    for (const auto& p : parts) {
      if (p.t.scalar_type() != at::kByte) type_error("the cache's ", p.name, " must be uint8, got ", p.t.scalar_type());
      if (p.t.sizes() != p.want || !p.t.is_contiguous() || (uintptr_t)p.t.const_data_ptr() % 16)
        value_error("the cache's ", p.name, " must be contiguous, 16-byte aligned ", dims(p.want), ", got ", dims(p.t.sizes()));
    }
    layer = integer("layer", args[4]);
    if (layer < 0 || layer >= l) value_error("layer ", layer, " of a cache of ", l, " layers");
    for (const auto& [name, t] : {std::pair<const char*, const Tensor&>{"table", table}, {"lens", lens}})
      if (t.scalar_type() != at::kInt) type_error(name, " must be int32, got ", t.scalar_type());
    if (lens.dim() != 1 || !lens.is_contiguous() || lens.size(0) < 1 || lens.size(0) > 65535)
      value_error("lens must be contiguous [sequences], 1 to 65535 of them, got ", dims(lens.sizes()), " / ", dims(lens.strides()));
    if (table.dim() != 2 || table.size(0) != lens.size(0) || table.size(1) < 1 || !unit_stride(table) || table.size(1) >= 1 << 25)
      value_error("table must be [", lens.size(0), ", pages of a sequence] with contiguous rows, got ", dims(table.sizes()), " / ",
                  dims(table.strides()));
    if (starts.defined() && starts.size(0) != lens.size(0) + 1)
      value_error("starts ", dims(starts.sizes()), " must be (", lens.size(0) + 1, ",) for ", lens.size(0), " sequences");
    same_device("KV4Cache", k4, ks, v4, vs, table, lens, starts);
  }
  int64_t seqs() const { return lens.size(0); }
  int64_t t_stride() const { return table.size(0) <= 1 ? 0 : table.stride(0); }
  const int32_t* first() const { return starts.defined() ? (const int32_t*)starts.data_ptr() : nullptr; }
  uint8_t* of(const Tensor& t) const { return (uint8_t*)t.data_ptr() + layer * (t.numel() / t.size(0)); }
  void check_rows(const char* name, int64_t n) {
    rows = n;
    if (!starts.defined() && n != seqs()) value_error(name, " has ", n, " rows for ", seqs(), " sequences: give starts");
    if (!k4.is_cuda()) value_error("the cache must be on a device (it has no CPU implementation)");
  }
  void same_heads(const char* name, const Tensor& t) const {
    if (t.size(2) != dim) value_error(name, " ", dims(t.sizes()), " does not have the cache's ", dim, " channels");
    same_device("KV4Cache", k4, t);
  }
};

}  // namespace

// The operator as users call it: the rotation's arguments, then q_weight, k_weight, eps. (q, k or None), with a gradient where
// one is recorded.
PyObject* norm_rotary_embed(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 12);
  const NormRotary a(args);
  if (!records_gradient(a.q, a.k, a.weight[0], a.weight[1])) return wrap_all(a.forward());
  const auto out = NormRotaryFunction::apply(a.q, maybe(a.k), maybe(a.weight[0]), maybe(a.weight[1]), &a);
  return wrap_all(std::array<Tensor, 2>{out[0], a.k.defined() ? out[1] : Tensor()});
  END_HANDLE_TH_ERRORS
}

// q, k, v, starts, k_starts, sm_scale, causal
PyObject* packed_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 7);
  const Packed a(args);
  if (!records_gradient(a.q, a.k, a.v)) return wrap(a.forward(nullptr));
  return wrap(PackedFunction::apply(a.q, a.k, a.v, &a));
  END_HANDLE_TH_ERRORS
}

// The cache's four parts, layer, table, lens, starts, k, v
PyObject* kv4_write(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 10);
  no_gradient("KV4Cache.write", args, n);
  Cache c(args);
  const Tensor &k = row_tensor("k", args[8]), &v = row_tensor("v", args[9]);
  if (k.sizes() != v.sizes() || k.size(1) != c.heads)
    value_error("k ", dims(k.sizes()), " and v ", dims(v.sizes()), " must be [rows, ", c.heads, ", ", c.dim, "]");
  if (k.scalar_type() != v.scalar_type()) type_error("k (", k.scalar_type(), ") and v (", v.scalar_type(), ") must have one dtype");
  c.same_heads("k", k);
  same_device("KV4Cache", k, v);
  c.check_rows("k", k.size(0));
  if (c.rows) {
    const On on(k);
    const Tensor kr = rows_of(k), vr = rows_of(v);
    done(lbw_kv4_write(kr.data_ptr(), vr.data_ptr(), half_format("k", k), c.seqs(), c.rows, c.heads, c.dim, tok_stride(kr), head_stride(kr),
                       tok_stride(vr), head_stride(vr), c.first(), (const int32_t*)c.lens.data_ptr(), (const int32_t*)c.table.data_ptr(),
                       c.t_stride(), c.table.size(1), c.pages, c.of(c.k4), c.of(c.ks), c.of(c.v4), c.of(c.vs), on.stream),
         "lbw_kv4_write");
    for (const Tensor& t : {c.k4, c.ks, c.v4, c.vs})
      if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// The cache's four parts, layer, table, lens, starts, rows (None: one for each sequence)
PyObject* kv4_read(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 9);
  Cache c(args);
  const int64_t rows = args[8] == Py_None ? c.seqs() : integer("tokens", args[8]);
  if (rows < 0 || rows >= int64_t(1) << 31) value_error("tokens must be 0 to 2^31 - 1, got ", rows);
  if (args[8] == Py_None && c.starts.defined()) value_error("with starts, say how many tokens there are");
  c.check_rows("the call", rows);
  const On on(c.k4);
  std::array<Tensor, 2> out;
  for (Tensor& t : out) t = at::empty({rows, c.heads, c.dim}, c.k4.options().dtype(at::kBFloat16));
  if (rows)
    done(lbw_kv4_read(c.seqs(), rows, c.heads, c.dim, c.first(), (const int32_t*)c.lens.data_ptr(), (const int32_t*)c.table.data_ptr(),
                      c.t_stride(), c.table.size(1), c.pages, c.of(c.k4), c.of(c.ks), c.of(c.v4), c.of(c.vs), out[0].data_ptr(),
                      out[1].data_ptr(), on.stream),
         "lbw_kv4_read");
  return wrap_all(out);
  END_HANDLE_TH_ERRORS
}

// The cache's four parts, layer, table, lens, starts, q, sm_scale
PyObject* kv4_attend(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 10);
  no_gradient("KV4Cache.attend", args, n);
  Cache c(args);
  const Tensor& q = row_tensor("q", args[8]);
  if (q.size(1) % c.heads) value_error(q.size(1), " heads of q cannot share ", c.heads, " of the cache evenly");
  const float scale = scale_of(args[9], q.size(2));
  c.same_heads("q", q);
  c.check_rows("q", q.size(0));
  Tensor out = new_like(q);
  if (c.rows) {
    const On on(q);
    const Tensor qr = rows_of(q);
    const int64_t bytes = lbw_kv4_attn_workspace_bytes(c.seqs(), c.rows, q.size(1), c.heads, c.dim, c.table.size(1), !c.starts.defined());
    const Tensor ws = bytes ? at::empty({bytes}, q.options().dtype(at::kByte)) : Tensor();
    done(lbw_kv4_attn(qr.data_ptr(), half_format("q", q), c.seqs(), c.rows, q.size(1), c.heads, c.dim, tok_stride(qr), head_stride(qr),
                      c.first(), (const int32_t*)c.lens.data_ptr(), (const int32_t*)c.table.data_ptr(), c.t_stride(), c.table.size(1),
                      c.pages, c.of(c.k4), c.of(c.ks), c.of(c.v4), c.of(c.vs), scale, out.data_ptr(), ptr(ws), on.stream),
         "lbw_kv4_attn");
  }
  return wrap(out);
  END_HANDLE_TH_ERRORS
}

}  // namespace lbw_py
